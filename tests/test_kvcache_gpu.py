"""Writing a cache of 8-bit keys and values and reading it back (csrc/kvcache.hip): bit for bit what the definition gives in 64 bits
(scales are powers of two: every value in between is exact, a code is one rounding)."""
import math

import pytest
import torch

import kv_plain
from vision_amd.kvcache import KVCache

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def rows_of(counts, H, D, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    n = sum(counts)
    x = torch.randn((n, H, D), generator=g) * torch.exp(spread * torch.randn((n, 1, 1), generator=g))
    return x.to(dtype)


def offsets_of(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


class Both:
    """The cache on the GPU beside the plain one, sequence by sequence and head by head."""

    def __init__(self, sequences, H, D, block, format, width=4, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.H, self.D, self.block = H, D, block
        self.table = torch.randperm(sequences * width + 2, generator=g)[:sequences * width].view(sequences, width).to(torch.int32)
        self.cache = KVCache(sequences * width + 2, H, D, block=block, format=format, device=DEV)
        self.plain = [[[kv_plain.Cache(block, format) for _ in range(H)] for _ in range(sequences)] for _ in "kv"]
        self.dev_table = self.table.to(DEV)

    def append(self, k, v, counts, start, **kw):
        off = offsets_of(counts)
        uniform = len(set(counts)) == 1 and off[-1] == k.shape[0] and kw.pop("uniform", True)
        self.cache.append(k.to(DEV), v.to(DEV), self.dev_table, i32(start), **({} if uniform else dict(offsets=i32(off))), **kw)
        for x, plain in zip((k, v), self.plain):
            for b, (o, s) in enumerate(zip(off, start)):
                room = self.table.shape[1] * self.block - s
                for h in range(self.H):
                    plain[b][h].append(x[o:o + min(counts[b], max(room, 0)), h].double(), s)

    def check(self, first, counts):
        off = offsets_of(counts)
        for dtype in (torch.float32, torch.bfloat16):
            got = self.cache.read(self.dev_table, i32(first), off[-1], offsets=i32(off), most=max(counts), dtype=dtype)
            for x, plain in zip(got, self.plain):
                for b, (o, n) in enumerate(zip(off, counts)):
                    want = torch.stack([plain[b][h].read(first[b], n, self.D) for h in range(self.H)], 1)
                    assert torch.equal(x[o:o + n].double().cpu().nan_to_num(nan=1e30), want.nan_to_num(nan=1e30)), (dtype, b)


CASES = [  # block, format, heads, dim
    (64, "e4m3", 2, 128), (64, "int8", 3, 64), (128, "e4m3", 1, 80), (128, "int8", 2, 16), (256, "e4m3", 1, 256), (256, "int8", 1, 48),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_prompts_tokens_and_read_back(case, dtype):
    block, format, H, D = case
    both = Both(3, H, D, block, format)
    prompt = [block + 5, 1, 2 * block]
    both.append(rows_of(prompt, H, D, dtype, 1), rows_of(prompt, H, D, dtype, 2), prompt, [0, 0, 0])
    both.check([0, 0, 0], prompt)
    at = list(prompt)
    for step in range(6):                                    # single tokens; the last sequence begins a block
        spread = 0.0 if step % 2 else 3.0                    # scales grow
        both.append(rows_of([1] * 3, H, D, dtype, 10 + step, spread), rows_of([1] * 3, H, D, dtype, 20 + step, spread), [1] * 3, at)
        at = [a + 1 for a in at]
        both.check([0, 0, 0], at)
    more = [block - 3, 70, 3]                                # from inside a block over its end
    both.append(rows_of(more, H, D, dtype, 5, 2.0), rows_of(more, H, D, dtype, 6, 2.0), more, at)
    at = [a + m for a, m in zip(at, more)]
    both.check([0, 0, 0], at)
    both.check([3, 1, block - 1], [1, 0, 2])                 # single rows, none, over a border


def test_rewriting_inside_a_block_keeps_its_other_tokens():
    both = Both(1, 2, 32, 64, "e4m3")
    both.append(rows_of([40], 2, 32, torch.float32, 1), rows_of([40], 2, 32, torch.float32, 2), [40], [0])
    big = rows_of([6], 2, 32, torch.float32, 3) * 100
    both.append(big, big * 3, [6], [9])                      # grows the scale: tokens before and behind move along
    both.check([0], [40])
    both.append(big / 1e4, big / 1e4, [2], [30])             # and does not shrink it
    both.check([0], [40])


def test_a_block_starts_anew():
    c = KVCache(1, 1, 16, device=DEV)
    t, zero = i32([[0]]), i32([0])
    x = torch.full((64, 1, 16), 300.0, device=DEV)
    c.append(x, x, t, zero)
    y = torch.full((2, 1, 16), 0.01171875, device=DEV)
    c.append(y, y, t, zero)
    k, _ = c.read(t, zero, 2, dtype=torch.float32)
    assert torch.equal(k, y)                                 # as fine as if nothing had been there


@pytest.mark.parametrize("format", ["e4m3", "int8"])
def test_values_at_the_borders(format):
    """Each extreme in a block of its own: zeros, denormals, the largest float, ties, magnitudes next to a scale's border."""
    top = kv_plain.LARGEST[format]
    vals = [0.0, 1e-45, 2.0 ** -126, 2.0 ** -110 * top, 2.0 ** -115, 3.4028234663852886e38, top, top * (1 + 2.0 ** -22), top * 2, 1.0,
            2.0 ** 100 * top, 1.9921875 * 2.0 ** 6, 2.0 ** -100]
    blocks = []
    for v in vals:
        row = torch.linspace(-1, 1, 64 * 16).view(64, 1, 16).double() * v
        row[0, 0, 0] = v
        blocks.append(row.float())
    both = Both(1, 1, 16, 64, format, width=len(vals))
    x = torch.cat(blocks)
    both.append(x, -x, [x.shape[0]], [0])
    both.check([0], [x.shape[0]])
    assert torch.isfinite(both.cache.read(both.dev_table, i32([0]), x.shape[0], dtype=torch.float32)[0]).all()


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("format", ["e4m3", "int8"])
def test_what_is_not_finite(bad, format):
    both = Both(2, 2, 32, 64, format)
    k, v = rows_of([70, 70], 2, 32, torch.float32, 1), rows_of([70, 70], 2, 32, torch.float32, 2)
    k[3, 1, 7] = bad                                         # sequence 0, head 1, first block of keys only
    both.append(k, v, [70, 70], [0, 0])
    both.check([0, 0], [70, 70])
    got = both.cache.read(both.dev_table, i32([0, 0]), 140, dtype=torch.float32)
    assert torch.isnan(got[0][:64, 1]).all() and torch.isfinite(got[0][:, 0]).all() and torch.isfinite(got[0][64:, 1]).all()
    assert torch.isfinite(got[1]).all()
    one = rows_of([1, 1], 2, 32, torch.float32, 3)
    both.append(one, one, [1, 1], [20, 20])                  # stays so while the block lives
    both.check([0, 0], [70, 70])
    both.append(one, one, [1, 1], [0, 0])                    # and is gone when it starts anew
    assert torch.isfinite(both.cache.read(both.dev_table, i32([0, 0]), 2, dtype=torch.float32)[0]).all()
    codes = both.cache.codes_k if format == "e4m3" else None
    assert codes is None or not ((codes & 127) == 127).any()  # no code is ever NaN


def test_a_value_that_is_not_finite_arrives_later():
    both = Both(1, 1, 16, 64, "e4m3")
    x = rows_of([10], 1, 16, torch.float32, 1)
    both.append(x, x, [10], [0])
    y = rows_of([1], 1, 16, torch.float32, 2)
    y[0, 0, 0] = math.inf
    both.append(y, x[:1], [1], [10])
    both.check([0], [11])


def test_holes_and_rows_that_belong_nowhere():
    H, D = 2, 32
    c = KVCache(4, H, D, device=DEV)
    table = i32([[0, -1, 2], [4, 1, 2147483647], [3, -2147483648, -1]])
    counts = [192, 130, 0]
    k = rows_of([322 + 20], H, D, torch.float32, 1).to(DEV)   # 20 rows behind the last sequence
    off = i32([0, 192, 322, 322])
    c.append(k, k, table, i32([0, 0, 0]), offsets=off)
    assert (c.scales_k[3] == 0).all() and (c.scales_k[:3] > 0).all()
    for dtype in (torch.float32, torch.bfloat16):
        mark = [torch.full((342, H, D), 7.0, dtype=dtype, device=DEV) for _ in "kv"]
        out = c.read(table, i32([0, 0, 0]), 342, offsets=off, out=mark)
        assert out[0] is mark[0]
        for x in out:
            assert (x[64:128] == 0).all() and (x[192:256] == 0).all() and (x[320:322] == 0).all() and (x[322:] == 7).all()
            assert (x[:64] != 0).any() and (x[128:192] != 0).any() and (x[256:320] != 0).any()
    # negative starts, rows behind the table, offsets of any content, `most` below a sequence's rows
    before = c.codes_k.clone(), c.scales_k.clone()
    c.append(k[:6], k[:6], table, i32([-1, -2147483648, 192]))
    c.append(k[:6], k[:6], table, i32([2147483647, 2147483640, 1000000]))
    c.append(k[:6], k[:6], table, i32([0, 0, 0]), offsets=i32([9, 3, -4, 2]), most=0)
    assert torch.equal(before[0], c.codes_k) and torch.equal(before[1], c.scales_k)
    mark = [torch.full((6, H, D), 7.0, device=DEV) for _ in "kv"]
    c.read(table, i32([-1, 0, 2147483647]), 6, out=mark)
    assert (mark[0][:2] == 7).all() and (mark[0][2:4] == 0).all() and (mark[0][4:] == 0).all()
    mark = [torch.full((6, H, D), 7.0, device=DEV) for _ in "kv"]
    c.read(table, i32([0, 0, 0]), 6, offsets=i32([0, 5, 5, 6]), most=2, out=mark)
    assert (mark[0][2:5] == 7).all() and (mark[0][5] != 7).all()


def test_strides_and_alignment():
    H, D, n = 3, 48, 100
    table = i32([[0, 1]])
    base = rows_of([n], H, D, torch.float32, 1)
    for dtype in (torch.float32, torch.bfloat16):
        x = base.to(dtype)
        want = None
        fused = torch.zeros((n, 3 * H * D + 1), dtype=dtype, device=DEV)
        fused[:, 1:1 + H * D] = x.flatten(1).to(DEV)
        fused[:, 1 + H * D:1 + 2 * H * D] = x.flatten(1).to(DEV)
        heads_first = x.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)
        spread = torch.zeros((n, H, 2 * D), dtype=dtype, device=DEV)
        spread[..., ::2] = x.to(DEV)
        for k in (x.to(DEV), fused[:, 1:1 + H * D].unflatten(1, (H, D)), heads_first, spread[..., ::2]):
            c = KVCache(2, H, D, device=DEV)
            c.append(k, k, table, i32([0]))
            got = c.codes_k, c.codes_v, c.scales_k, c.scales_v
            assert want is None or all(torch.equal(a, b) for a, b in zip(want, got))
            want = got
        c = KVCache(2, H, D, device=DEV)
        one = x[:1].to(DEV).expand(n, H, D)                  # one row for every token
        c.append(one, one, table, i32([0]))
        k, v = c.read(table, i32([0]), n, dtype=dtype)
        assert (k == k[:1]).all()
        out = torch.zeros((n, 2, H * D + 1), dtype=dtype, device=DEV)[:, :, 1:].unflatten(2, (H, D))
        c.read(table, i32([0]), n, out=(out[:, 0], out[:, 1]))
        assert torch.equal(out[:, 0], k) and torch.equal(out[:, 1], v)


def test_long_cache():
    """Blocks whose bytes lie behind 2^32."""
    H, D, block = 8, 256, 256
    blocks = 2 ** 32 // (H * D * block) + 3
    c = KVCache(blocks, H, D, block=block, device=DEV)
    table = i32([[blocks - 1, 1], [blocks - 2, 0]])
    k, v = rows_of([300, 300], H, D, torch.bfloat16, 1).to(DEV), rows_of([300, 300], H, D, torch.bfloat16, 2).to(DEV)
    c.append(k, v, table, i32([0, 0]))
    small = KVCache(4, H, D, block=block, device=DEV)
    t2 = i32([[0, 1], [2, 3]])
    small.append(k, v, t2, i32([0, 0]))
    for a, b in zip(c.read(table, i32([0, 0]), 600), small.read(t2, i32([0, 0]), 600)):
        assert torch.equal(a, b)


def test_streams_and_graphs():
    """A decoding loop captured once: positions advance on the device, the cache is written and read by every replay."""
    H, D = 2, 64
    a, b = KVCache(4, H, D, device=DEV), KVCache(4, H, D, device=DEV)
    table = i32([[0, 1], [2, 3]])
    k, v = rows_of([2], H, D, torch.bfloat16, 1).to(DEV), rows_of([2], H, D, torch.bfloat16, 2).to(DEV)
    start, zero = i32([60, 0]), i32([0, 0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.append(k, v, table, start)
        got = a.read(table, zero, 130, offsets=OFF, most=70)
        start += 1
    a.codes_k.zero_(), a.codes_v.zero_(), a.scales_k.zero_(), a.scales_v.zero_()
    start.copy_(i32([60, 0]))
    for step in range(8):
        k.copy_(rows_of([2], H, D, torch.bfloat16, 30 + step)), v.copy_(rows_of([2], H, D, torch.bfloat16, 60 + step))
        graph.replay()
        b.append(k, v, table, i32([60 + step, step]))
        want = b.read(table, zero, 130, offsets=OFF, most=70)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want, got)), step
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.append(k, v, table, start)
        got = b.read(table, zero, 130, offsets=OFF, most=70)
    torch.cuda.current_stream().wait_stream(side)
    a.append(k, v, table, start)
    assert all(torch.equal(x, y) for x, y in zip(a.read(table, zero, 130, offsets=OFF, most=70), got))


OFF = None


@pytest.fixture(autouse=True)
def _offsets():
    global OFF
    OFF = i32([0, 70, 130])


def test_refuses_a_cache_on_another_device():
    c = KVCache(2, 1, 16, device=DEV)
    x = torch.zeros(1, 1, 16)
    with pytest.raises(ValueError, match="is on"):
        c.append(x, x, i32([[0]]), i32([0]))
    with pytest.raises(ValueError, match="is on"):
        c.append(x.to(DEV), x.to(DEV), torch.zeros(1, 1, dtype=torch.int32), i32([0]))
