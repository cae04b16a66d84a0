"""Attention over the 8-bit cache: how many bits a result keeps where there are few queries (all but its own rounding), and queries that are
one row in memory for many tokens."""
import pytest
import torch

import kv_plain
from test_kv_attention_gpu import filled, i32, offsets_of, rnd
from vision_amd import _lib
from vision_amd._lib import lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(2, 4, 128, 64, "e4m3"), (3, 1, 64, 64, "int8"), (1, 5, 256, 256, "e4m3"), (2, 2, 192, 64, "int8"), (1, 8, 80, 128, "e4m3")],
                         ids=lambda s: "x".join(map(str, s)))
def test_bf16_probabilities_keep_sixteen_bits(shape):
    H, G, D, block, format = shape
    lengths, counts = [1, 2, 49, 64, 65, 300, 2000, 9000], [1, 2, 3, 1, 2, 1, 1, 1]
    c, table, k, v, off = filled(lengths, H, D, block, format, 5)
    q = rnd((sum(counts), H * G, D), torch.bfloat16, 9)
    out = c.attend(q, table, i32(lengths), offsets=i32(offsets_of(counts)), most=3).double().cpu()
    qo = offsets_of(counts)
    for b, (n, L) in enumerate(zip(counts, lengths)):
        want, size, reach = kv_plain.attend(q[qo[b]:qo[b + 1]], k[off[b]:off[b + 1]], v[off[b]:off[b + 1]], L, D ** -0.5)
        # as kv_plain.attend_bound, but a probability is the sum of two bf16 numbers: 2^-8 of 2^-8
        u = 2.0 ** -24
        rel = 2 * (D + 4) * u * reach + 2 * (L + L / 32 + 16) * u
        bound = 2.0 ** -8 * want.abs() + (1 + 2.0 ** -8) * (2.0 ** -16 + rel) * size + 1e-30
        worst = ((out[qo[b]:qo[b + 1]] - want).abs() / bound).max()
        assert worst <= 1, (b, L, float(worst))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("H,count", [(2, 1), (2, 50), (16, 70), (16, 200)])
def test_expanded_queries(H, count, dtype):
    """One row of queries for every token (a token stride of 0): every row is that of the same queries laid out; small and large tiles."""
    D = 48
    lengths = [250, 201]
    c, table, k, v, off = filled(lengths, H, D, 64, "e4m3", 360)
    t = _lib.F32 if dtype == torch.float32 else _lib.BF16
    sequences = [0, 1] * (1 if H == 2 else 8)
    tile = lib.vamd_kv_attend_tile(count * len(sequences), len(sequences), count, 250, H, 3, D, 0, 0, t)
    assert tile == (16 if H == 2 else 128)
    one = rnd((1, 3 * H, D), dtype, 369).expand(count * len(sequences), 3 * H, D)
    lengths, table = i32([lengths[b] for b in sequences]), table[sequences].contiguous()
    for kw in ({}, dict(window=30, sinks=2), dict(causal=False)):
        out = c.attend(one, table, lengths, longest=250, **kw)
        assert torch.equal(out, c.attend(one.contiguous(), table, lengths, longest=250, **kw))
    # without the causal bound all tokens of a sequence see the same
    assert torch.equal(out.view(len(sequences), count, 3 * H, D), out.view(len(sequences), count, 3 * H, D)[:, :1].expand(-1, count, -1, -1))
