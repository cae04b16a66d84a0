"""Attention over the 8-bit cache (csrc/kv_attention.hip) against its formula in 64 bits on what the cache reads back (that is
exact and has tests of its own); the bound of each element's error is derived in kv_plain.attend_bound."""
import math

import pytest
import torch

import kv_plain
from vision_amd import _lib
from vision_amd._lib import lib
from vision_amd.kvcache import KVCache
from vision_amd.rotary import Rotary

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def rnd(shape, dtype, seed, spread=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    if spread:
        x = x * torch.exp(spread * torch.randn((shape[0], 1, 1), generator=g)) * torch.exp(spread * torch.randn((1,) + tuple(shape[1:]), generator=g))
    return x.to(dtype).to(DEV)


def offsets_of(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def filled(lengths, H, D, block, format, seed=0, spread=0.4, width=None):
    """A cache with sequences of these lengths, its table, and its keys and values as read back."""
    width = width or max(1, max((n + block - 1) // block for n in lengths))
    B = len(lengths)
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(B * width + 3, generator=g)[:B * width].view(B, width).to(torch.int32).to(DEV)
    c = KVCache(B * width + 3, H, D, block=block, format=format, device=DEV)
    off = offsets_of(lengths)
    if off[-1]:
        c.append(rnd((off[-1], H, D), torch.bfloat16, seed + 1, spread), rnd((off[-1], H, D), torch.bfloat16, seed + 2, spread), table,
                 i32([0] * B), offsets=i32(off), most=max(lengths))
    k, v = c.read(table, i32([0] * B), off[-1], offsets=i32(off), most=max(lengths) if off[-1] else 0, dtype=torch.float32)
    return c, table, k.cpu(), v.cpu(), off


def compare(out, q, k, v, off, lengths, counts, scale, dtype, holes=None, **kw):
    qo = offsets_of(counts)
    out = out.double().cpu()
    for b, (n, L) in enumerate(zip(counts, lengths)):
        D = q.shape[2]
        want, size, reach = kv_plain.attend(q[qo[b]:qo[b + 1]], k[off[b]:off[b + 1]], v[off[b]:off[b + 1]], L, scale,
                                            holes=None if holes is None else holes[b], **kw)
        bound = kv_plain.attend_bound(want, size, reach, L, D, dtype)
        got = out[qo[b]:qo[b + 1]]
        worst = ((got - want).abs() / bound).max() if n else 0
        assert not torch.isnan(got).any() and worst <= 1, (b, n, L, float(worst))


DTYPES = [torch.bfloat16, torch.float32]
SHAPES = [  # kv heads, group, dim, block, format
    (2, 4, 128, 64, "e4m3"), (3, 1, 64, 64, "int8"), (1, 8, 80, 128, "int8"), (2, 3, 16, 64, "e4m3"), (1, 5, 256, 256, "e4m3"),
    (1, 16, 96, 64, "int8"), (1, 17, 48, 128, "e4m3"), (2, 2, 192, 64, "int8"), (1, 40, 112, 64, "e4m3"),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_single_tokens(shape, dtype):
    H, G, D, block, format = shape
    lengths = [1, 2, 63, 64, 65, 130, 257, 700, 0]
    c, table, k, v, off = filled(lengths, H, D, block, format)
    q = rnd((len(lengths), H * G, D), dtype, 9)
    out = c.attend(q, table, i32(lengths))
    compare(out, q, k, v, off, lengths, [1] * len(lengths), D ** -0.5, dtype)
    assert (out[-1] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_prompts(shape, dtype):
    H, G, D, block, format = shape
    lengths, counts = [1, 70, 200, 333, 5, 64, 129], [1, 70, 3, 150, 0, 64, 66]
    c, table, k, v, off = filled(lengths, H, D, block, format, 20)
    n = sum(counts)
    q = rnd((n + 5, H * G, D), dtype, 29)
    out = torch.full_like(q, 7.0)
    got = c.attend(q, table, i32(lengths), offsets=i32(offsets_of(counts)), most=max(counts), scale=0.3, out=out)
    assert got is out and (out[n:] == 7).all()               # rows of no sequence are left as they were
    compare(out, q, k, v, off, lengths, counts, 0.3, dtype)
    again = c.attend(q[:n], table, i32(lengths), offsets=i32(offsets_of(counts)), scale=0.3)
    assert torch.equal(again, out[:n])                       # without `most`
    full = c.attend(q[:n], table, i32(lengths), offsets=i32(offsets_of(counts)), most=max(counts), causal=False)
    compare(full, q, k, v, off, lengths, counts, D ** -0.5, dtype, causal=False)


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (64, 0), (65, 4), (100, 64), (100, 65), (500, 3), (5000, 2), (17, 300), (30, 2 ** 31 - 1)])
def test_window_and_sinks(window, sinks, dtype):
    lengths, counts = [1, 64, 333, 700, 901], [1, 64, 100, 1, 130]
    c, table, k, v, off = filled(lengths, 2, 64, 64, "e4m3", 40)
    q = rnd((sum(counts), 6, 64), dtype, 49)
    out = c.attend(q, table, i32(lengths), offsets=i32(offsets_of(counts)), most=max(counts), window=window, sinks=sinks)
    compare(out, q, k, v, off, lengths, counts, 0.125, dtype, window=window, sinks=sinks)
    if sinks == 2 ** 31 - 1:
        assert torch.equal(out, c.attend(q, table, i32(lengths), offsets=i32(offsets_of(counts)), most=max(counts), window=window, sinks=2 ** 32 + 1))
    one = c.attend(q[:5], table, i32(lengths), window=window, sinks=sinks)
    compare(one, q[:5], k, v, off, lengths, [1] * 5, 0.125, dtype, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("format", ["e4m3", "int8"])
def test_long_contexts_split_and_joined(format, dtype):
    lengths = [20000, 513, 6001]
    c, table, k, v, off = filled(lengths, 1, 128, 128, format, 60)
    q = rnd((3, 4, 128), dtype, 69)
    assert lib.vamd_kv_attend_workspace(3, 3, 1, 20000, 1, 4, 128, 0, 0, _lib.BF16) > 0
    out = c.attend(q, table, i32(lengths), longest=20000)
    compare(out, q, k, v, off, lengths, [1, 1, 1], 128 ** -0.5, dtype)
    # the bound steers the split only: too low, or far too high, the result is right
    for longest in (1, 700, 5000, 10 ** 9):
        compare(c.attend(q, table, i32(lengths), longest=longest), q, k, v, off, lengths, [1, 1, 1], 128 ** -0.5, dtype)
    q = rnd((60, 4, 128), dtype, 70)
    compare(c.attend(q, table, i32(lengths)), q, k, v, off, lengths, [20] * 3, 128 ** -0.5, dtype)
    w = c.attend(q, table, i32(lengths), window=3000, sinks=70)
    compare(w, q, k, v, off, lengths, [20] * 3, 128 ** -0.5, dtype, window=3000, sinks=70)


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
def test_many_short_sequences_without_most(dtype):
    """Rows of unlike number, none known to the host: few tiles, split along the keys and joined."""
    counts = [1, 0, 2, 9, 1, 1, 5, 0, 3] * 9
    lengths = [(700 * i) % 4001 + 9 for i in range(len(counts))]
    c, table, k, v, off = filled(lengths, 1, 64, 64, "e4m3", 75)
    q = rnd((sum(counts), 6, 64), dtype, 79)
    assert lib.vamd_kv_attend_workspace(sum(counts), len(counts), sum(counts), table.shape[1] * 64, 1, 6, 64, 0, 0, _lib.BF16) > 0
    for window in (0, 1500):
        out = c.attend(q, table, i32(lengths), offsets=i32(offsets_of(counts)), window=window, sinks=5)
        compare(out, q, k, v, off, lengths, counts, 0.125, dtype, **(dict(window=window, sinks=5) if window else {}))


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
def test_many_queries(dtype):
    """Prompts of many tiles, behind an earlier context, windowed or not."""
    lengths, counts = [700, 1100], [700, 600]
    c, table, k, v, off = filled(lengths, 2, 128, 64, "e4m3", 80)
    q = rnd((1300, 4, 128), dtype, 89)
    o = i32(offsets_of(counts))
    compare(c.attend(q, table, i32(lengths), offsets=o, most=700), q, k, v, off, lengths, counts, 128 ** -0.5, dtype)
    compare(c.attend(q, table, i32(lengths), offsets=o, most=700, window=200, sinks=5), q, k, v, off, lengths, counts, 128 ** -0.5, dtype,
            window=200, sinks=5)


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("count", [1, 90])
def test_holes(dtype, count):
    lengths = [300, 300, 64]
    c, table, k, v, off = filled(lengths, 2, 64, 64, "int8", 100)
    table = table.clone()
    table[0, 1], table[0, 4], table[1, 0], table[2, 0] = -1, c.blocks, 2147483647, -7
    holes = [torch.zeros(320, dtype=torch.bool) for _ in lengths]
    holes[0][64:128] = holes[0][256:320] = holes[1][:64] = True
    holes[2][:64] = True
    q = rnd((3 * count, 4, 64), dtype, 109)
    out = c.attend(q, table, i32(lengths))
    compare(out, q, k, v, off, lengths, [count] * 3, 0.125, dtype, holes=holes)
    assert (out[2 * count:] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
def test_more_queries_than_tokens(dtype):
    """Queries before position 0 see nothing; lengths beyond the table are cut, negative ones are empty."""
    lengths = [3, 40, 64]
    c, table, k, v, off = filled(lengths, 1, 32, 64, "e4m3", 120)
    q = rnd((3 * 30, 2, 32), dtype, 129)
    out = c.attend(q, table, i32(lengths))
    compare(out, q, k, v, off, lengths, [30] * 3, 32 ** -0.5, dtype)
    assert (out[:27] == 0).all()
    cut = c.attend(q, table, i32([-5, 40, 2147483647]))
    assert (cut[:30] == 0).all() and torch.equal(cut[30:], out[30:])


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("count", [1, 40])
def test_what_is_not_finite(dtype, count):
    """A block that reads as NaN is NaN to the queries that see a token of it, and to no other."""
    c, table, k, v, off = filled([200, 200], 2, 64, 64, "e4m3", 140)
    clean = rnd((2 * count, 4, 64), dtype, 149)
    want = c.attend(clean, table, i32([200, 200]), window=72, sinks=3)
    bad = torch.full((1, 2, 64), math.nan, device=DEV)
    c.append(bad, bad, table[:1], i32([70]))                  # block 1 (tokens 64 .. 127) of sequence 0
    out = c.attend(clean, table, i32([200, 200]), window=72, sinks=3)
    assert torch.equal(out[count:], want[count:])
    first = 200 - count + torch.arange(count) - 71            # first token of each query's window
    for i in range(count):
        assert torch.isnan(out[i]).all() if first[i] < 128 else torch.equal(out[i], want[i]), i
    # what lies behind the last token is not seen: NaN in a later block, stale codes in the same one
    c2, table2, *_ = filled([64], 1, 64, 64, "int8", 150, width=2)
    q = rnd((1, 1, 64), dtype, 151)
    one = c2.attend(q, table2, i32([64]))
    c2.append(torch.full((64, 1, 64), math.inf, device=DEV), torch.full((64, 1, 64), math.nan, device=DEV), table2, i32([64]))
    assert torch.equal(c2.attend(q, table2, i32([64])), one)
    # queries that are not finite concern their own rows only
    clean[0, 0, 0] = math.nan
    mixed = c.attend(clean, table, i32([200, 200]), window=1)
    assert torch.isnan(mixed[0, 0]).all() and torch.isfinite(mixed[0, 1:]).all() and torch.isfinite(mixed[1:]).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
def test_large_scores(dtype):
    """Scores of several thousand and one dominant key per query: the running maximum moves at every step."""
    L, D = 260, 64
    c = KVCache(5, 1, D, device=DEV)
    table = i32([[0, 1, 2, 3, 4]])
    k = torch.zeros(L, 1, D, device=DEV)
    k[:, 0, 0] = torch.arange(L, device=DEV) * 8.0
    v = rnd((L, 1, D), torch.float32, 1)
    c.append(k, v, table, i32([0]))
    kb, vb = c.read(table, i32([0]), L, dtype=torch.float32)
    q = torch.zeros(2, 2, D, dtype=dtype, device=DEV)
    q[0, 0, 0], q[0, 1, 0], q[1, 0, 0], q[1, 1, 0] = 16.0, -16.0, 0.03125, 300.0
    out = c.attend(q, table, i32([L]), causal=False)
    compare(out, q, kb.cpu(), vb.cpu(), [0, L], [L], [2], 0.125, dtype, causal=False)
    zero = c.attend(q, table, i32([L]), scale=0.0, causal=False)
    compare(zero, q, kb.cpu(), vb.cpu(), [0, L], [L], [2], 0.0, dtype, causal=False)
    negative = c.attend(q, table, i32([L]), scale=-0.01, causal=False)
    compare(negative, q, kb.cpu(), vb.cpu(), [0, L], [L], [2], -0.01, dtype, causal=False)


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("count", [1, 50])
def test_strides_alignment_and_in_place(dtype, count):
    H, G, D = 2, 3, 48
    lengths = [150, 90]
    c, table, k, v, off = filled(lengths, H, D, 64, "e4m3", 160)
    n = 2 * count
    q = rnd((n, H * G, D), dtype, 169)
    want = c.attend(q, table, i32(lengths))
    compare(want, q, k, v, off, lengths, [count] * 2, D ** -0.5, dtype)
    fused = torch.zeros((n, 2 * H * G * D + 1), dtype=dtype, device=DEV)
    view = fused[:, 1:1 + H * G * D].unflatten(1, (H * G, D))
    view.copy_(q)
    out = fused[:, 1 + H * G * D:].unflatten(1, (H * G, D))
    c.attend(view, table, i32(lengths), out=out)
    assert torch.equal(out, want) and torch.equal(view, q)
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.zeros((H * G, n, D), dtype=dtype, device=DEV).transpose(0, 1)
    assert torch.equal(c.attend(heads_first, table, i32(lengths), out=out), want)
    wide = torch.zeros((n, H * G, 2 * D), dtype=dtype, device=DEV)
    wide[..., ::2] = q
    assert torch.equal(c.attend(wide[..., ::2], table, i32(lengths)), want)
    same = q.clone()
    assert c.attend(same, table, i32(lengths), out=same) is same and torch.equal(same, want)
    one = q[:1].expand(n, H * G, D)
    assert torch.equal(c.attend(one, table, i32(lengths))[0], want[0]) or count > 1


# ---------------------------------------------------------------------------------------------------- large tiles
# (what the sizes above do not reach: 64 or 128 rows a workgroup, where a call is large enough)

def tile_of(rows, sequences, most, longest, H, G, D, dtype, window=0, sinks=0):
    return lib.vamd_kv_attend_tile(rows, sequences, most, longest, H, G, D, window, sinks, _lib.F32 if dtype == torch.float32 else _lib.BF16)


def batch_of(tile, longest, most, H, G, D, dtype, even=False):
    """Lengths and query counts of the smallest batch of this kind that is served by tiles of `tile` rows; unequal, one sequence
    without queries, one that ends with a group, unless `even`."""
    g = torch.Generator().manual_seed(D + G)
    lengths = torch.randint(1, longest + 1, (400,), generator=g).tolist()
    counts = [min(n, int(m)) for n, m in zip(lengths, torch.randint(0, most + 1, (400,), generator=g))]
    lengths[0], counts[0] = longest, most
    lengths[1], counts[1] = 64, min(64, most)
    counts[2] = 0
    if even:
        lengths, counts = [longest] * 400, [most] * 400
    for n in range(4, 400):
        if tile_of(sum(counts[:n]), n, most, longest, H, G, D, dtype) == tile:
            return lengths[:n], counts[:n]
    raise AssertionError("no such batch")


def attend_large(tile, c, q, table, lengths, counts, G, dtype, window=0, sinks=0, **kw):
    longest, most = max(lengths), max(counts)
    assert tile_of(q.shape[0], len(lengths), most, longest, c.kv_heads, G, c.head_dim, dtype, window, sinks) == tile
    return c.attend(q, table, i32(lengths), offsets=i32(offsets_of(counts)), most=most, longest=longest, window=window, sinks=sinks, **kw)


TILES = pytest.mark.parametrize("tile", [64, 128])


@TILES
@pytest.mark.parametrize("format", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, d) for d in (16, 32, 48, 64, 80, 96, 112, 128, 160, 176, 192, 224, 256)] +
                         [(torch.float32, d) for d in (16, 32, 48, 64, 80, 96, 112, 128)], ids=lambda x: str(x).replace("torch.", ""))
def test_large_tiles(dtype, D, format, tile):
    H = 16
    lengths, counts = batch_of(tile, 150, 130, H, 1, D, dtype)
    c, table, k, v, off = filled(lengths, H, D, 64, format, 220)
    q = rnd((sum(counts), H, D), dtype, 229)
    compare(attend_large(tile, c, q, table, lengths, counts, 1, dtype), q, k, v, off, lengths, counts, D ** -0.5, dtype)


@TILES
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("group", [1, 3, 8])
def test_large_tiles_groups_windows_and_edges(group, dtype, tile):
    H, D = 12, 64
    lengths, counts = batch_of(tile, 260, 80, H, group, D, dtype)
    c, table, k, v, off = filled(lengths, H, D, 128, "e4m3", 240)
    n = sum(counts)
    q = rnd((n + 3, H * group, D), dtype, 249)
    out = torch.full_like(q, 7.0)
    attend_large(tile, c, q, table, lengths, counts, group, dtype, out=out)
    assert (out[n:] == 7).all()
    compare(out, q, k, v, off, lengths, counts, 0.125, dtype)
    for window, sinks in ((1, 0), (64, 4), (100, 70), (1000, 3)) if group < 8 else ((64, 4),):
        compare(attend_large(tile, c, q, table, lengths, counts, group, dtype, window, sinks), q, k, v, off, lengths, counts, 0.125, dtype,
                window=window, sinks=sinks)
    if group == 8:
        return
    compare(attend_large(tile, c, q, table, lengths, counts, group, dtype, causal=False, scale=-0.2), q, k, v, off, lengths, counts, -0.2,
            dtype, causal=False)
    zero = attend_large(tile, c, q, table, lengths, counts, group, dtype, scale=0.0)
    compare(zero, q, k, v, off, lengths, counts, 0.0, dtype)
    # more queries than tokens, lengths of zero, beyond the table and negative
    odd = [0, -3] + [2 ** 31 - 1 if i % 7 == 0 else max(1, n // 3) for i, n in enumerate(lengths[2:])]
    got = c.attend(q[:n], table, i32(odd), offsets=i32(offsets_of(counts)), most=max(counts))
    room = table.shape[1] * c.block
    kr, vr = c.read(table, i32([0] * len(odd)), room * len(odd), dtype=torch.float32)
    compare(got, q, kr.cpu(), vr.cpu(), [room * b for b in range(len(odd) + 1)], [min(max(x, 0), room) for x in odd], counts, 0.125, dtype)


@TILES
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
def test_large_tiles_holes_and_what_is_not_finite(dtype, tile):
    H, G, D = 16, 2, 32
    lengths, counts = batch_of(tile, 300, 40, H, G, D, dtype, even=True)
    count = len(lengths)
    c, table, k, v, off = filled(lengths, H, D, 64, "e4m3", 260)
    q = rnd((40 * count, H * G, D), dtype, 269)
    clean = attend_large(tile, c, q, table, lengths, counts, G, dtype, window=72, sinks=3)
    bad = torch.full((1, H, D), math.nan, device=DEV)
    c.append(bad, bad, table[:1], i32([200]))                 # block 3 (tokens 192 .. 255) of sequence 0
    out = attend_large(tile, c, q, table, lengths, counts, G, dtype, window=72, sinks=3)
    assert torch.equal(out[40:], clean[40:])
    for i in range(40):                                       # query 260 + i sees tokens from 189 + i on
        assert torch.isnan(out[i]).all() if 189 + i < 256 else torch.equal(out[i], clean[i]), i
    table = table.clone()
    table[0, 3], table[1, 0], table[2, 4], table[3] = -1, c.blocks, 2 ** 31 - 1, -5
    holes = [torch.zeros(320, dtype=torch.bool) for _ in lengths]
    holes[0][192:256] = holes[1][:64] = holes[2][256:] = holes[3][:] = True
    out = attend_large(tile, c, q, table, lengths, counts, G, dtype)
    compare(out, q, k, v, off, lengths, counts, 32 ** -0.5, dtype, holes=holes)
    assert (out[120:160] == 0).all()


@TILES
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
def test_large_tiles_values_of_any_scale(dtype, tile):
    """Values' scales far from 1 (they go into the probabilities' exponent while that is safe), zero blocks, blocks of unlike scale."""
    H, D = 16, 32
    lengths, counts = batch_of(tile, 256, 70, H, 1, D, dtype, even=True)
    n = len(lengths)
    c = KVCache(4 * n, H, D, device=DEV)
    table = torch.arange(4 * n, dtype=torch.int32, device=DEV).view(n, 4)
    k, v = rnd((256 * n, H, D), torch.float32, 1), rnd((256 * n, H, D), torch.float32, 2).view(n, 4, 64, H, D)
    for b in range(n):
        for i in range(4):
            v[b, i] *= (2.0 ** -90, 2.0 ** 60, 0.0, 1.0, 2.0 ** -45, 2.0 ** 45, 2.0 ** 100)[(b + 3 * i) % 7] if b else (0.0, 1.0, 0.0, 2.0 ** -100)[i]
    c.append(k, v.view(-1, H, D), table, i32([0] * n))
    kb, vb = c.read(table, i32([0] * n), 256 * n, dtype=torch.float32)
    q = rnd((70 * n, H, D), dtype, 3)
    out = attend_large(tile, c, q, table, lengths, counts, 1, dtype)
    compare(out, q, kb.cpu(), vb.cpu(), [256 * b for b in range(n + 1)], lengths, counts, D ** -0.5, dtype)


@pytest.mark.parametrize("tile,longest", [(64, 11000), (128, 16000)])
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
def test_large_tiles_split_and_joined(dtype, tile, longest):
    H, G, D = 8, 2, 64
    lengths, counts = [longest, 9000, 40, 1500, 5000, 700], [40, 64, 40, 1, 33, 0]
    c, table, k, v, off = filled(lengths, H, D, 64, "int8", 280)
    q = rnd((sum(counts), H * G, D), dtype, 289)
    t = _lib.F32 if dtype == torch.float32 else _lib.BF16
    assert lib.vamd_kv_attend_workspace(sum(counts), 6, 64, longest, H, G, D, 0, 0, t) > 0
    compare(attend_large(tile, c, q, table, lengths, counts, G, dtype), q, k, v, off, lengths, counts, 0.125, dtype)
    compare(attend_large(tile, c, q, table, lengths, counts, G, dtype, longest - 100, 70), q, k, v, off, lengths, counts, 0.125, dtype, window=longest - 100,
            sinks=70)
    want = attend_large(tile, c, q, table, lengths, counts, G, dtype)
    g = torch.cuda.CUDAGraph()
    n, o = i32(lengths), i32(offsets_of(counts))
    with torch.cuda.graph(g):
        got = c.attend(q, table, n, offsets=o, most=64, longest=longest)
    for step in range(3):
        g.replay()
        assert torch.equal(c.attend(q, table, n, offsets=o, most=64, longest=longest), want)
        torch.cuda.synchronize()
        assert torch.equal(got, want), step


@TILES
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
def test_large_tiles_strides_and_in_place(dtype, tile):
    H, D = 16, 48
    lengths, counts = batch_of(tile, 90, 70, H, 1, D, dtype, even=True)
    c, table, k, v, off = filled(lengths, H, D, 64, "e4m3", 300)
    n = sum(counts)
    q = rnd((n, H, D), dtype, 309)
    want = attend_large(tile, c, q, table, lengths, counts, 1, dtype)
    compare(want, q, k, v, off, lengths, counts, D ** -0.5, dtype)
    fused = torch.zeros((n, 2 * H * D + 1), dtype=dtype, device=DEV)
    view, out = fused[:, 1:1 + H * D].unflatten(1, (H, D)), fused[:, 1 + H * D:].unflatten(1, (H, D))
    view.copy_(q)
    c.attend(view, table, i32(lengths), longest=90, out=out)
    assert torch.equal(out, want) and torch.equal(view, q)
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(c.attend(heads_first, table, i32(lengths), longest=90), want)
    same = q.clone()
    assert c.attend(same, table, i32(lengths), longest=90, out=same) is same and torch.equal(same, want)


@pytest.mark.parametrize("H,most", [(1, 80), (2, 80), (4, 80), (2, 20)])
def test_many_sequences(H, most):
    """More sequences than a wave has lanes: whose tile a workgroup takes is found 64 sequences at a time; tiles of any size."""
    count, D = 150, 32
    lengths = [1 + (37 * i) % 90 for i in range(count)]
    counts = [0 if i % 5 == 0 else min(n, 1 + (i * 13) % most) for i, n in enumerate(lengths)]
    counts[149], lengths[149] = most, 90
    c, table, k, v, off = filled(lengths, H, D, 64, "e4m3", 320)
    q = rnd((sum(counts), H, D), torch.bfloat16, 329)
    assert tile_of(sum(counts), count, most, 90, H, 1, D, torch.bfloat16) == {(1, 80): 16, (2, 80): 64, (4, 80): 128, (2, 20): 16}[H, most]
    out = c.attend(q, table, i32(lengths), offsets=i32(offsets_of(counts)), most=most, longest=90)
    compare(out, q, k, v, off, lengths, counts, D ** -0.5, torch.bfloat16)


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("sequences,H", [(3, 2), (50, 16)])
def test_rows_beyond_most_are_left_out(dtype, sequences, H):
    """... and the others keep their positions; small and large tiles."""
    lengths, counts, most = [200] * sequences, [90 - i % 3 * 40 for i in range(sequences)], 70
    c, table, k, v, off = filled(lengths, H, 32, 64, "e4m3", 340)
    o = offsets_of(counts)
    q = rnd((o[-1], H, 32), dtype, 349)
    assert tile_of(o[-1], sequences, most, 200, H, 1, 32, dtype) == (16 if sequences == 3 else 128)
    want = c.attend(q, table, i32(lengths), offsets=i32(o), most=max(counts), longest=200)
    got = c.attend(q, table, i32(lengths), offsets=i32(o), most=most, longest=200, out=torch.full_like(q, 7.0))
    compare(want, q, k, v, off, lengths, counts, 32 ** -0.5, dtype)
    for b, n in enumerate(counts):
        assert torch.allclose(got[o[b]:o[b] + min(n, most)].float(), want[o[b]:o[b] + min(n, most)].float(), atol=2e-2, rtol=2e-2)
        assert (got[o[b] + min(n, most):o[b + 1]] == 7).all()


def test_no_rows():
    c, table, *_ = filled([10], 1, 32, 64, "e4m3", 170)
    assert c.attend(torch.zeros(0, 2, 32, device=DEV), table, i32([10])).shape == (0, 2, 32)


def test_same_result_every_time():
    lengths = [5000, 300]
    c, table, k, v, off = filled(lengths, 2, 128, 64, "e4m3", 180)
    q = rnd((2, 8, 128), torch.bfloat16, 189)
    want = c.attend(q, table, i32(lengths))
    for _ in range(5):
        assert torch.equal(c.attend(q, table, i32(lengths)), want)


def test_streams():
    """Two calls at once on two streams: each has its own workspace."""
    lengths = [9000, 300]
    c, table, k, v, off = filled(lengths, 2, 64, 64, "e4m3", 190)
    q = [rnd((2, 8, 64), torch.bfloat16, 191 + i) for i in range(2)]
    want = [c.attend(x, table, i32(lengths)) for x in q]
    n = i32(lengths)
    streams = [torch.cuda.Stream() for _ in q]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(c.attend(q[i], table, n))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


def test_two_graphs():
    """Two captured graphs of split calls, replayed in turn with eager work between; lengths advance on the device."""
    lengths = [9000, 2000]
    c, table, k, v, off = filled([9100, 2100], 2, 64, 64, "int8", 200)
    n = i32(lengths)
    q = [rnd((2, 8, 64), torch.bfloat16, 201 + i) for i in range(2)]
    graphs, outs = [], []
    for x in q:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.attend(x, table, n, window=0))
        graphs.append(g)
    for step in range(4):
        for i in (0, 1, 0):
            q[i].copy_(rnd((2, 8, 64), torch.bfloat16, 300 + step * 3 + i))
            n.copy_(i32([9000 + step, 2000 + 20 * step]))
            graphs[i].replay()
            eager = c.attend(q[i], table, n)
            torch.cuda.synchronize()
            assert torch.equal(outs[i], eager), (step, i)


def test_decoding_as_it_is_used():
    """A prompt and then single tokens: positions turned, the cache written, attention over it; against 64 bits on the turned
    queries and the values the cache reads back."""
    H, G, D, steps = 2, 2, 64, 12
    for dtype in DTYPES:
        r = Rotary(D, 48, scaling={"type": "ntk", "factor": 2.0}, device=DEV)
        c = KVCache(8, H, D, device=DEV)
        table = i32([[0, 5, 2], [7, 1, 3]])
        counts, at = [60, 20], [0, 0]
        for step in range(steps):
            n = sum(counts)
            q, k, v = (rnd((n, h, D), dtype, 10 * step + i) for i, h in enumerate((H * G, H, H)))
            positions = torch.cat([torch.arange(a, a + m) for a, m in zip(at, counts)]).to(DEV)
            o = i32(offsets_of(counts))
            q, k = r(positions, q, k)
            c.append(k, v, table, i32(at), offsets=o, most=max(counts))
            at = [a + m for a, m in zip(at, counts)]
            out = c.attend(q, table, i32(at), offsets=o, most=max(counts))
            off = offsets_of(at)
            kb, vb = c.read(table, i32([0, 0]), off[-1], offsets=i32(off), most=max(at), dtype=torch.float32)
            compare(out, q, kb.cpu(), vb.cpu(), off, at, counts, D ** -0.5, dtype)
            counts = [1, 1]
        # what 8 bits cost: e4m3 keeps 4 significant bits of the last step's keys
        err = (kb[off[1] - 1] - k[0].float()).abs() / k[0].float().abs().clamp(min=0.05)
        assert err.max() <= 2.0 ** -4


def test_long_cache():
    """Blocks whose bytes lie behind 2^32."""
    H, D, block = 8, 256, 256
    blocks = 2 ** 32 // (H * D * block) + 3
    c = KVCache(blocks, H, D, block=block, device=DEV)
    table = i32([[blocks - 1, 1], [blocks - 2, 0]])
    k, v = rnd((600, H, D), torch.bfloat16, 1, 0.4), rnd((600, H, D), torch.bfloat16, 2, 0.4)
    c.append(k, v, table, i32([0, 0]))
    kb, vb = c.read(table, i32([0, 0]), 600, dtype=torch.float32)
    for n in (1, 40):
        q = rnd((2 * n, H, D), torch.bfloat16, 3)
        compare(c.attend(q, table, i32([300, 300])), q, kb.cpu(), vb.cpu(), [0, 300, 600], [300, 300], [n, n], 0.0625, torch.bfloat16)
