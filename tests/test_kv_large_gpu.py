"""Calls of the rotary positions, the 8-bit cache and the attention over it that are large in their number of workgroups."""
import pytest
import torch

from vision_amd.kvcache import KVCache
from vision_amd.rotary import Rotary

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def test_rotary_of_more_than_2_to_32_lanes():
    n, r = 1_500_000_000, Rotary(6, 2, device=DEV)           # three lanes a token
    q = torch.zeros(n, 1, 6, dtype=torch.bfloat16, device=DEV)
    at = i32([0, 1, n // 3, n // 2, 1431655765, 1431655766, n - 2, n - 1]).long()
    q[at] = 1
    pos = torch.ones(n, dtype=torch.int32, device=DEV)
    r.apply_(pos, q)
    want = r(pos[:1], torch.ones(1, 1, 6, dtype=torch.bfloat16, device=DEV))
    assert (want[..., :2] != 1).all() and torch.equal(q[at], want.expand(8, 1, 6))


def test_append_and_read_of_more_than_2_to_32_threads():
    """Prompts whose longest is not known to the host."""
    B, rows, H, D, block = 300, 1 << 17, 16, 16, 64
    counts = [(rows // B) + (-1) ** b * (b % 97) for b in range(B)]
    counts[-1] += rows - sum(counts)
    offsets = [0]
    for c in counts:
        offsets.append(offsets[-1] + c)
    width = (max(counts) + block - 1) // block
    assert B * (rows // block) * 2 * H > 1 << 24             # by sequences and rows, 256 threads each
    table = torch.randperm(B * width, device=DEV).to(torch.int32).view(B, width)
    k, v = torch.randn(rows, H, D, device=DEV).bfloat16(), torch.randn(rows, H, D, device=DEV).bfloat16()
    zero, off = torch.zeros(B, dtype=torch.int32, device=DEV), i32(offsets)
    caches = [KVCache(B * width, H, D, block=block, device=DEV) for _ in range(2)]
    caches[0].append(k, v, table, zero, offsets=off)
    caches[1].append(k, v, table, zero, offsets=off, most=max(counts))
    for name in ("codes_k", "codes_v", "scales_k", "scales_v"):
        assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), name
    for a, b, x in zip(caches[0].read(table, zero, rows, offsets=off), caches[1].read(table, zero, rows, offsets=off, most=max(counts)), (k, v)):
        assert torch.equal(a, b)
        assert ((a.float() - x.float()).abs() <= x.float().abs() * 2.0 ** -4 + 2.0 ** -16).all()     # half a step; scales are 2^-6 at most


def test_attention_of_more_than_2_to_32_threads():
    B, H, D = (1 << 20) + 3, 16, 16
    c = KVCache(2, H, D, device=DEV)
    k = torch.randn(40, H, D, device=DEV)
    c.append(k, k.flip(0), i32([[1]]), i32([0]))
    table, lengths = torch.ones(B, 1, dtype=torch.int32, device=DEV), torch.full((B,), 40, dtype=torch.int32, device=DEV)
    q = torch.randn(7, H, D, device=DEV).bfloat16()
    out = c.attend(q[torch.arange(B, device=DEV) % 7], table, lengths)
    want = c.attend(q, table[:7], lengths[:7])
    assert torch.equal(out, want[torch.arange(B, device=DEV) % 7])


@pytest.mark.parametrize("block", [64, 256])
def test_append_and_read_go_by_the_rows_there_are(block):
    """Many ragged prompts of unknown length: by sequences times rows this call would not fit into any launch."""
    B, H, D = 4096, 12, 16
    counts = [(b * 37) % 1024 if b % 5 else 0 for b in range(B)]
    starts = [-1 if b % 11 == 10 else (b * 13) % 100 for b in range(B)]
    rows = sum(counts) + 9                                   # nine that belong to no sequence
    offsets = [0]
    for c in counts:
        offsets.append(offsets[-1] + c)
    assert B * (rows // block) * 2 * H > 2 ** 31 or block == 256
    width = (1024 + 100 + block - 1) // block + 1
    table = torch.randperm(B * width, device=DEV).to(torch.int32).view(B, width)
    k, v = torch.randn(rows, H, D, device=DEV), torch.randn(rows, H, D, device=DEV)
    off, start = i32(offsets), i32(starts)
    caches = [KVCache(B * width, H, D, block=block, format="int8", device=DEV) for _ in range(2)]
    caches[0].append(k, v, table, start, offsets=off)
    caches[1].append(k, v, table, start, offsets=off, most=max(counts))
    for name in ("codes_k", "codes_v", "scales_k", "scales_v"):
        assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), name
    out = [tuple(torch.full((rows, H, D), 7.0, device=DEV) for _ in "kv") for _ in caches]
    caches[0].read(table, start, rows, offsets=off, out=out[0])
    caches[1].read(table, start, rows, offsets=off, most=max(counts), out=out[1])
    assert all(torch.equal(a, b) for a, b in zip(*out))
    owned = torch.cat([torch.full((c,), s >= 0) for c, s in zip(counts, starts)] + [torch.zeros(9, dtype=torch.bool)]).to(DEV)
    assert (out[0][0][~owned] == 7).all() and (out[0][0][owned] != 7).any(1).any(1).all()
    few = caches[0].read(table, start, rows, offsets=off, most=3, out=tuple(torch.full((rows, H, D), 7.0, device=DEV) for _ in "kv"))
    at = torch.cat([torch.arange(c) for c in counts] + [torch.full((9,), 9)]).to(DEV)
    assert torch.equal(few[0], torch.where((at < 3)[:, None, None], out[0][0], 7.0))
