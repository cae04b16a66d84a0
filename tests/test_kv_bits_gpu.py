"""How many bits attention over the 8-bit cache keeps where there are few queries: all but the result's own rounding."""
import pytest
import torch

import kv_plain
from test_kv_attention_gpu import filled, i32, offsets_of, rnd

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
