"""Attention over cached values up to the largest float (csrc/kv_attention.hip): the result is a mean of values, finite as they are, for
every tile size, split or not.  Formula and bound as in test_kv_attention_gpu.py."""
import pytest
import torch

import kv_plain
from test_kv_attention_gpu import DEV, DTYPES, attend_large, batch_of, compare, i32, offsets_of, rnd
from vision_amd import _lib
from vision_amd._lib import lib
from vision_amd.kvcache import KVCache

pytestmark = pytest.mark.gpu


def filled(lengths, H, D, format, exponents, seed, rise):
    """Scores that rise with the position (by `rise` in all, in powers of e, for a query of ones); block i of a sequence has values of
    2^exponents[i], some of one sign throughout, so that sums of them would pass the largest float."""
    B, width = len(lengths), (max(lengths) + 63) // 64
    c = KVCache(B * width, H, D, format=format, device=DEV)
    table = torch.randperm(B * width, generator=torch.Generator().manual_seed(seed)).view(B, width).to(torch.int32).to(DEV)
    off = offsets_of(lengths)
    k, v = rnd((off[-1], H, D), torch.float32, seed + 1) * 0.02, rnd((off[-1], H, D), torch.float32, seed + 2)
    at = torch.cat([torch.arange(n) for n in lengths]).to(DEV)
    k += (rise * D ** -0.5 * at / max(lengths))[:, None, None]
    v = v.clamp(-1.9, 1.9)
    v[..., ::3] = v[..., ::3].abs()
    v[..., 1::3] = 1.9 - v[..., 1::3].abs() * 0.05
    v = torch.ldexp(v, torch.tensor(exponents, dtype=torch.int32, device=DEV)[at // 64 % len(exponents)][:, None, None])
    assert torch.isfinite(v).all()
    c.append(k, v, table, i32([0] * B), offsets=i32(off), most=max(lengths))
    kb, vb = c.read(table, i32([0] * B), off[-1], offsets=i32(off), most=max(lengths), dtype=torch.float32)
    assert torch.isfinite(vb).all()
    return c, table, kb.cpu(), vb.cpu(), off


RANGES = [(127,), (126, 120, 127, 110), (0, 127, -60, 126), (40, 41, 48, 49, 50)]


@pytest.mark.parametrize("exponents", RANGES, ids=str)
@pytest.mark.parametrize("format", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
def test_few_queries(dtype, format, exponents):
    H, G, D = 2, 3, 64
    lengths, counts = [700, 64, 333, 1], [5, 1, 9, 1]
    c, table, k, v, off = filled(lengths, H, D, format, exponents, 10, 6.0)
    q = rnd((sum(counts), H * G, D), dtype, 13) * 0.1 + 1
    compare(c.attend(q, table, i32(lengths), offsets=i32(offsets_of(counts)), most=9), q, k, v, off, lengths, counts, D ** -0.5, dtype)
    one = c.attend(q[:4], table, i32(lengths))
    compare(one, q[:4], k, v, off, lengths, [1] * 4, D ** -0.5, dtype)


@pytest.mark.parametrize("exponents", RANGES, ids=str)
@pytest.mark.parametrize("format", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("tile", [64, 128])
def test_large_tiles(tile, dtype, format, exponents):
    H, D = 16, 32
    lengths, counts = batch_of(tile, 400, 70, H, 1, D, dtype)
    c, table, k, v, off = filled(lengths, H, D, format, exponents, 20, 7.0)
    q = rnd((sum(counts), H, D), dtype, 23) * 0.1 + 1
    compare(attend_large(tile, c, q, table, lengths, counts, 1, dtype), q, k, v, off, lengths, counts, D ** -0.5, dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
def test_split_and_joined(dtype):
    D = 64
    lengths = [20000, 6001]
    c, table, k, v, off = filled(lengths, 1, D, "e4m3", (127, 126, -30, 127), 30, 9.0)
    t = _lib.F32 if dtype == torch.float32 else _lib.BF16
    q = rnd((2, 4, D), dtype, 33) * 0.1 + 1
    assert lib.vamd_kv_attend_workspace(2, 2, 1, 20000, 1, 4, D, 0, 0, t) > 0
    compare(c.attend(q, table, i32(lengths)), q, k, v, off, lengths, [1, 1], D ** -0.5, dtype)
    H, G, counts = 8, 2, [40, 64]
    lengths = [11000, 9000]
    c, table, k, v, off = filled(lengths, H, D, "int8", (127, 126, -30, 127), 40, 9.0)
    q = rnd((sum(counts), H * G, D), dtype, 43) * 0.1 + 1
    assert lib.vamd_kv_attend_workspace(sum(counts), 2, 64, 11000, H, G, D, 0, 0, t) > 0
    assert lib.vamd_kv_attend_tile(sum(counts), 2, 64, 11000, H, G, D, 0, 0, t) in (16, 64, 128)
    compare(c.attend(q, table, i32(lengths), offsets=i32(offsets_of(counts)), most=64, longest=11000), q, k, v, off, lengths, counts, D ** -0.5, dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
def test_small_values_beside_large_ones_that_are_not_seen(dtype):
    """A row that does not see the large block, or gives it no weight, keeps its small values."""
    D, H = 64, 1
    c = KVCache(3, H, D, device=DEV)
    table = i32([[0, 1, 2]])
    k = torch.zeros(192, H, D, device=DEV)
    k[64:128, :, 0] = -100.0                                 # the second block: values of 2^127, weight 0 to the first query head
    v = rnd((192, H, D), torch.float32, 5)
    v[:64] *= 2.0 ** -100
    v[64:128] = 2.0 ** 127
    v[128:] *= 2.0 ** -100
    c.append(k, v, table, i32([0]))
    kb, vb = c.read(table, i32([0]), 192, dtype=torch.float32)
    for n in (1, 60, 140):
        q = torch.zeros(n, 2, D, dtype=dtype, device=DEV)
        q[:, 0, 0], q[:, 1, 0] = 300.0, 0.5
        out = c.attend(q, table, i32([192]))
        compare(out, q, kb.cpu(), vb.cpu(), [0, 192], [192], [n], D ** -0.5, dtype)
        assert (out[:, 0].abs() < 2.0 ** -90).all() and (out[:, 0] != 0).any()
