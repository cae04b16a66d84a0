"""Rotary positions, the 8-bit cache and attention over it: what can be checked without a GPU.  Refusals of the Python layer and of
the C entry points (they come before any device work), the frequencies, the index functions of csrc/kv_layout.h compiled for
the host, and the plain forms the GPU tests compare with."""
import copy
import ctypes
import math
import os
import random
import subprocess

import numpy as np
import pytest
import torch

import kv_plain
from conftest import ROOT
from vision_amd import _lib
from vision_amd._lib import lib
from vision_amd.kvcache import KVCache
from vision_amd.rotary import Rotary, rotary_frequencies


# ---------------------------------------------------------------------------------------------------- rotary

def test_frequencies():
    f, a = rotary_frequencies(8)
    assert a == 1.0 and f == [10000.0 ** (-i / 8) for i in (0, 2, 4, 6)]
    assert rotary_frequencies(8, 100.0, {"type": "linear", "factor": 4})[0] == [100.0 ** (-i / 8) / 4 for i in (0, 2, 4, 6)]
    f, a = rotary_frequencies(64, scaling={"type": "ntk", "factor": 8})
    plain = rotary_frequencies(64)[0]
    assert f[0] == plain[0] and math.isclose(f[-1], plain[-1] / 8, rel_tol=1e-12) and a == 1.0
    f, a = rotary_frequencies(64, scaling={"type": "yarn", "factor": 4, "original": 4096})
    for x, y in zip(f, plain):
        turns = 4096 * y / (2 * math.pi)
        want = y if turns >= 32 else y / 4 if turns <= 1 else None
        assert want is None or x == want
        assert y / 4 <= x <= y
    assert a == 0.1 * math.log(4) + 1
    # 64-bit fractions of a turn: positions up to 2^31 keep 30 bits of the angle
    r = Rotary(64, scaling={"type": "yarn", "factor": 4, "original": 4096})
    for bits, x in zip(r.frequencies.tolist(), f):
        assert abs((bits % 2 ** 64) / 2 ** 64 - x / (2 * math.pi)) <= 2.0 ** -53
    assert "frequencies" not in r.state_dict()


@pytest.mark.parametrize("bad", [dict(head_dim=64, rotary_dim=66), dict(head_dim=64, rotary_dim=7), dict(head_dim=64, rotary_dim=0),
                                 dict(head_dim=64, layout="other"), dict(head_dim=64, base=1.0), dict(head_dim=64, base=math.nan),
                                 dict(head_dim=64, scaling={"type": "other", "factor": 2}),
                                 dict(head_dim=64, scaling={"type": "linear", "factor": 0.5}),
                                 dict(head_dim=64, scaling={"type": "linear", "factor": 2, "original": 5}),
                                 dict(head_dim=64, scaling={"type": "yarn", "factor": 2, "original": 9, "alpha": 5, "beta": 4})])
def test_rotary_constructor_refuses(bad):
    with pytest.raises(ValueError):
        Rotary(**bad)


def test_rotary_missing_scaling_key():
    for scaling in ({"type": "linear"}, {"type": "yarn", "factor": 2}):
        with pytest.raises(KeyError):
            Rotary(64, scaling=scaling)


def test_rotary_call_refuses():
    r = Rotary(32)
    pos, q, k = torch.arange(5), torch.zeros(5, 4, 32), torch.zeros(5, 2, 32)
    with pytest.raises(TypeError):
        r(pos, q.half())
    with pytest.raises(TypeError):
        r(pos.float(), q)
    with pytest.raises(ValueError):
        r(pos, torch.zeros(5, 4, 16))
    with pytest.raises(ValueError):
        r(pos, q, k[:4])
    with pytest.raises(ValueError):
        r(pos, q, k.bfloat16())
    with pytest.raises(ValueError):
        r(pos[:4], q)
    with pytest.raises(ValueError):
        r(torch.zeros(2, 5, dtype=torch.int64), q)
    with pytest.raises(RuntimeError, match="GPU only"):
        r(pos, q, k)


P = 1 << 20                                                    # never followed: these calls fail before any launch


def rotary_call(**change):
    a = dict(positions=P, wide=1, frequencies=P, amplitude=1.0, batch=1, tokens=4, dim=32, turned=32, interleaved=0, inverse=0, q=P, yq=P,
             q_heads=2, qb=256, qt=64, qh=32, yb=256, yt=64, yh=32, k=None, yk=None, k_heads=0, kb=0, kt=0, kh=0, ykb=0, ykt=0, ykh=0, dtype=0)
    a.update(change)
    return lib.vamd_rotary(*a.values(), None)


@pytest.mark.parametrize("bad", [dict(positions=None), dict(q=None), dict(yq=None), dict(frequencies=None), dict(dim=1), dict(turned=3),
                                 dict(turned=34), dict(turned=0), dict(dtype=2), dict(q=P + 2), dict(positions=P + 4), dict(tokens=-1),
                                 dict(batch=-1), dict(q_heads=-1), dict(k_heads=2), dict(batch=2 ** 31 - 1, tokens=2 ** 20)])
def test_rotary_entry_refuses(bad):
    assert rotary_call(**bad) < 0 and b"vamd_rotary" in lib.vamd_last_error()


def test_rotary_entry_with_nothing_to_do():
    assert rotary_call(tokens=0) == 0 and rotary_call(q_heads=0) == 0 and rotary_call(batch=0) == 0


# ---------------------------------------------------------------------------------------------------- cache

@pytest.mark.parametrize("bad", [dict(block=32), dict(block=96), dict(head_dim=24), dict(head_dim=272), dict(head_dim=0), dict(blocks=0),
                                 dict(kv_heads=0), dict(format="e5m2")])
def test_cache_constructor_refuses(bad):
    with pytest.raises(ValueError):
        KVCache(**{**dict(blocks=2, kv_heads=2, head_dim=32, device="cpu"), **bad})


def _call(method, **change):
    c = KVCache(4, 2, 32, device="cpu")
    i32 = torch.int32
    a = dict(table=torch.zeros(2, 2, dtype=i32), offsets=None, most=None)
    if method == "append":
        a.update(k=torch.zeros(2, 2, 32), v=torch.zeros(2, 2, 32), start=torch.zeros(2, dtype=i32))
    elif method == "read":
        a.update(start=torch.zeros(2, dtype=i32), rows=2)
    else:
        a.update(q=torch.zeros(2, 6, 32), lengths=torch.ones(2, dtype=i32))
    a.update(change)
    return getattr(c, method)(**a)


@pytest.mark.parametrize("method", ["append", "read", "attend"])
def test_cache_runs_on_the_gpu_only(method):
    with pytest.raises(RuntimeError, match="GPU only"):
        _call(method)


def _i32(*n):
    return torch.zeros(n, dtype=torch.int32)


@pytest.mark.parametrize("method,error,bad", [
    ("append", TypeError, lambda: dict(k=torch.zeros(2, 2, 32).half())),
    ("append", ValueError, lambda: dict(k=torch.zeros(2, 3, 32))),
    ("append", ValueError, lambda: dict(k=torch.zeros(3, 2, 32))),
    ("append", ValueError, lambda: dict(k=torch.zeros(2, 2, 32).bfloat16())),
    ("append", ValueError, lambda: dict(k=torch.zeros(3, 2, 32), v=torch.zeros(3, 2, 32))),       # 3 rows, 2 sequences
    ("append", ValueError, lambda: dict(table=torch.zeros(2, 2, dtype=torch.int64))),
    ("append", ValueError, lambda: dict(table=_i32(2, 0))),
    ("append", ValueError, lambda: dict(table=_i32(2))),
    ("append", ValueError, lambda: dict(table=_i32(2, 4)[:, ::2])),
    ("append", ValueError, lambda: dict(start=_i32(3))),
    ("append", ValueError, lambda: dict(start=torch.zeros(2, dtype=torch.int64))),
    ("append", ValueError, lambda: dict(start=_i32(4)[::2])),
    ("append", ValueError, lambda: dict(offsets=_i32(2))),
    ("append", ValueError, lambda: dict(offsets=_i32(3), most=-1)),
    ("append", ValueError, lambda: dict(most=2)),
    ("append", RuntimeError, lambda: dict(k=torch.zeros(2, 2, 32, requires_grad=True))),
    ("read", TypeError, lambda: dict(dtype=torch.float16)),
    ("read", ValueError, lambda: dict(rows=3)),
    ("read", ValueError, lambda: dict(rows=-2)),
    ("read", ValueError, lambda: dict(out=(torch.zeros(2, 2, 32), torch.zeros(2, 2, 32).bfloat16()))),
    ("read", ValueError, lambda: dict(out=(torch.zeros(2, 2, 32), torch.zeros(1, 2, 32).expand(2, 2, 32)))),
    ("read", ValueError, lambda: dict(out=(torch.zeros(2, 2, 32),) * 2)),
    ("read", ValueError, lambda: (lambda x: dict(out=(x[:2], x[1:])))(torch.zeros(3, 2, 32))),
    ("read", ValueError, lambda: dict(out=(torch.zeros(2, 2, 64)[..., ::2], torch.zeros(2, 2, 32)))),
    ("attend", ValueError, lambda: dict(q=torch.zeros(2, 5, 32))),
    ("attend", ValueError, lambda: dict(q=torch.zeros(2, 0, 32))),
    ("attend", ValueError, lambda: dict(q=torch.zeros(2, 64))),
    ("attend", TypeError, lambda: dict(q=torch.zeros(2, 6, 32).double())),
    ("attend", ValueError, lambda: dict(window=-1)),
    ("attend", ValueError, lambda: dict(sinks=-1)),
    ("attend", ValueError, lambda: dict(window=4, causal=False)),
    ("attend", ValueError, lambda: dict(out=torch.zeros(2, 6, 16))),
    ("attend", ValueError, lambda: dict(out=torch.zeros(2, 6, 32).bfloat16())),
    ("attend", RuntimeError, lambda: dict(q=torch.zeros(2, 6, 32, requires_grad=True))),
    ("attend", ValueError, lambda: dict(lengths=_i32(1))),
])
def test_cache_call_refuses(method, error, bad):
    with pytest.raises(error) as e:
        _call(method, **bad())
    assert "GPU only" not in str(e.value)


def test_attend_refuses_overlapping_out():
    x = torch.zeros(3, 6, 32)
    with pytest.raises(ValueError, match="share memory"):
        _call("attend", q=x[:2], out=x[1:])


def test_overlapping_tells_exactly():
    import itertools
    rng, buf, seen = random.Random(1), torch.zeros(400), [0, 0]

    def places(t):
        return {t.storage_offset() + sum(i * s for i, s in zip(at, t.stride())) for at in itertools.product(*map(range, t.shape))}

    for _ in range(1500):
        dims = rng.randint(1, 4)
        strides = [rng.choice((0, 1, 1, 2, 3, 4, 5, 8, 12, 16, 24)) for _ in range(dims)]
        a, b = (buf.as_strided([rng.randint(1, 4) for _ in range(dims)], strides, rng.randint(0, 60)) for _ in range(2))
        if rng.random() < 0.5:
            b = buf.as_strided(b.shape, [rng.choice((0, 1, 2, 3, 7, 16)) for _ in range(dims)], b.storage_offset())
        want = bool(places(a) & places(b))
        seen[want] += 1
        assert _lib.overlapping(a, b) == want == _lib.overlapping(b, a), (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
    assert min(seen) > 300
    x = torch.zeros(4, 3, 12, 16)                           # queries and keys of one buffer, heads before or behind the tokens
    for y in (x, x.transpose(1, 2).contiguous().transpose(1, 2)):
        assert not _lib.overlapping(y[:, :, :8], y[:, :, 8:10]) and _lib.overlapping(y[:, :, :8], y[:, :, 7:9])
    assert not _lib.overlapping(x, x.clone()) and not _lib.overlapping(x[:0], x)


def test_a_copied_cache_is_its_own():
    c = KVCache(4, 2, 32, device="cpu")
    d = copy.deepcopy(c)
    assert not set(c._pool()) & set(d._pool()) and d._pool()[0] == d.codes_k.data_ptr()


def io_call(name, **change):
    a = dict(ck=P, cv=P, sk=P, sv=P, table=P, stride=2, start=P, offsets=None, rows=2, sequences=2, most=1, heads=2, dim=32, block=64, width=2,
             blocks=4, format=0, x=P, xt=64, xh=32, y=P, yt=64, yh=32, dtype=0)
    a.update(change)
    v = a.copy()
    if name == "vamd_kv_append":
        order = "x xt xh y yt yh ck cv sk sv table stride start offsets rows sequences most heads dim block width blocks format dtype"
    else:
        order = "ck cv sk sv table stride start offsets rows sequences most heads dim block width blocks format x xt xh y yt yh dtype"
    return getattr(lib, name)(*(v[n] for n in order.split()), None)


@pytest.mark.parametrize("name", ["vamd_kv_append", "vamd_kv_read"])
@pytest.mark.parametrize("bad", [dict(ck=None), dict(sv=None), dict(table=None), dict(start=None), dict(x=None), dict(y=None), dict(ck=P + 8),
                                 dict(x=P + 1), dict(dim=20), dict(dim=512), dict(block=32), dict(format=2), dict(dtype=3), dict(rows=3),
                                 dict(rows=-1, offsets=P), dict(most=-1), dict(heads=0), dict(sequences=0), dict(width=0), dict(blocks=0),
                                 dict(sequences=1 << 20, most=1 << 16, rows=1 << 36), dict(start=P + 2)])
def test_io_entries_refuse(name, bad):
    assert io_call(name, **bad) < 0 and name.encode() in lib.vamd_last_error()


@pytest.mark.parametrize("name", ["vamd_kv_append", "vamd_kv_read"])
def test_io_entries_with_nothing_to_do(name):
    assert io_call(name, rows=0, most=0) == 0


def attend_call(**change):
    a = dict(q=P, qt=64, qh=32, ck=P, cv=P, sk=P, sv=P, table=P, stride=2, lengths=P, offsets=None, rows=2, sequences=2, most=1, longest=128,
             heads=2, group=1, dim=32, block=64, width=2, blocks=4, format=0, scale=1.0, causal=1, window=0, sinks=0, o=P, ot=64, oh=32,
             work=None, size=0, dtype=0)
    a.update(change)
    return lib.vamd_kv_attend(*a.values(), None)


@pytest.mark.parametrize("bad", [dict(q=None), dict(o=None), dict(cv=None), dict(sk=None), dict(table=None), dict(lengths=None), dict(q=P + 2),
                                 dict(dim=8), dict(dim=288), dict(block=63), dict(format=-1), dict(dtype=7), dict(window=-1), dict(sinks=-1),
                                 dict(window=2, causal=0), dict(rows=3), dict(heads=0), dict(group=0), dict(width=0), dict(blocks=0),
                                 dict(width=2 ** 30), dict(most=2 ** 30, group=4, rows=2 ** 31), dict(most=2 ** 28 + 1, rows=2 ** 29 + 2), dict(longest=1 << 20),   # workspace needed, none given
                                 dict(longest=1 << 20, work=P + 8, size=1 << 40), dict(lengths=P + 1)])
def test_attend_entry_refuses(bad):
    assert attend_call(**bad) < 0 and b"vamd_kv_attend" in lib.vamd_last_error()


def test_attend_entry_with_nothing_to_do():
    assert attend_call(rows=0, most=0) == 0
    assert lib.vamd_kv_attend_workspace(1, 0, 1, 64, 1, 1, 64, 0, 0, 0) == 0


def test_attend_workspace_goes_by_the_rows_there_are():
    """However many rows a sequence might have by `most`: a share per workgroup, of which there are about as many as the chip holds."""
    for sequences, rows, heads, group, longest in [(255, 510, 1, 8, 1 << 20), (500, 500, 1, 4, 1 << 16), (100, 100, 2, 16, 1 << 18), (3, 900, 1, 1, 1 << 20),
                                                   (40, 1200, 2, 8, 1 << 20)]:
        for dim in (64, 256):
            for most in (1, rows // sequences + 1, rows):
                tile = lib.vamd_kv_attend_tile(rows, sequences, most, longest, heads, group, dim, 0, 0, _lib.BF16)
                size = lib.vamd_kv_attend_workspace(rows, sequences, most, longest, heads, group, dim, 0, 0, _lib.BF16)
                assert size <= 1024 * tile * (dim + 2) * 4, (sequences, rows, most, dim, size)


def test_attend_tiles_go_by_the_rows_there_are():
    def tile(rows, sequences, most, heads=8, group=4, dim=128):
        return lib.vamd_kv_attend_tile(rows, sequences, most, 4096, heads, group, dim, 0, 0, _lib.BF16)
    for heads, group, dim in [(8, 4, 128), (1, 8, 256), (4, 2, 64)]:         # two queries each, whether that is known or not
        assert tile(510, 255, 2, heads, group, dim) == tile(510, 255, 510, heads, group, dim) == 16
    assert tile(5021, 2, 4096) == tile(5021, 2, 5021) == tile(4096 + 63, 64, 4096) == 128       # prompts, with decoding steps beside them
    assert tile(800, 4, 200) == tile(800, 4, 800) == 64


# ---------------------------------------------------------------------------------------------------- index functions, on the host

HOST = r'''
#include <stdio.h>
#include <stdlib.h>
#include <set>
#include "kv_layout.h"
using namespace vamd;
int main(int argc, char** argv) {
    // every byte of a group has one place
    for (int D = 16; D <= 256; D += 16) {
        std::set<int> k, v;
        for (int t = 0; t < 64; ++t) for (int d = 0; d < D; ++d) { k.insert(kv_key_at(t, d, D)); v.insert(kv_value_at(t, d)); }
        if ((int)k.size() != 64 * D || *k.begin() != 0 || *k.rbegin() != 64 * D - 1) return 1;
        if ((int)v.size() != 64 * D || *v.begin() != 0 || *v.rbegin() != 64 * D - 1) return 2;
    }
    // tables and offsets of any content
    int32_t table[12] = {0, 3, -1, 4, 2147483647, -2147483647, 1, 2, 0, 0, 0, 0};
    const int want[6] = {0, 3, -1, -1, -1, -1};
    for (int i = 0; i < 6; ++i) if (kv_page(table, 6, 6, 4, 0, i) != want[i]) return 3;
    if (kv_page(table, 6, 6, 4, 1, 0) != 1 || kv_page(table, 6, 6, 4, 1, 6) != -1 || kv_page(table, 6, 6, 4, 0, -1) != -1 ||
        kv_page(table, 6, 6, 4, 0, 1ll << 40) != -1) return 4;
    const int32_t off[6] = {-5, 3, 2, 100, 2147483647, 7};
    for (int b = 0; b < 5; ++b) for (int most = 0; most < 12; ++most) {
        const KvRows r = kv_rows(off, b, 10, most);
        if (r.first < 0 || r.count < 0 || r.count > most || r.first + r.count > 10 || r.all < r.count || r.first + r.all > 10) return 5;
    }
    if (kv_rows(NULL, 3, 20, 5).first != 15 || kv_rows(NULL, 3, 20, 5).count != 5) return 6;
    // every row of a call falls into one span; a negative start into none
    for (int unit = 64; unit <= 256; unit *= 2) for (int start = 0; start < 300; start += 7) for (int n = 0; n < 600; n += 11) {
        int rows = 0, touched = n ? (n + unit - 2) / unit + 1 : 0;
        for (int j = 0; j < touched; ++j) {
            const KvSpan s = kv_span(start, n, (start / unit + j) * (int64_t)unit, unit);
            if (s.lo < 0 || s.lo > unit || s.hi > unit) return 7;
            if (s.hi > s.lo) rows += s.hi - s.lo;
        }
        if (rows != n) return 8;
        const KvSpan s = kv_span(-1 - start, n, 0, unit);
        if (s.hi > s.lo) return 9;
    }
    if (kv_span(2147483647, 5, 2147483584ll, 64).hi != 64 || kv_span(2147483647, 5, 2147483584ll, 64).lo != 63) return 10;
    // scales: argv floats -> bits
    for (int i = 1; i < argc; ++i) {
        const uint32_t b = (uint32_t)strtoul(argv[i], NULL, 16);
        printf("%08x %08x\n", kv_scale_bits<VAMD_KV_E4M3>(b), kv_scale_bits<VAMD_KV_INT8>(b));
    }
    return 0;
}
'''


def test_index_functions_on_the_host(tmp_path):
    src = tmp_path / "host.hip"
    src.write_text(HOST)
    exe = str(tmp_path / "host")
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "--offload-host-only", "-O1", "-std=c++17", "-I",
                    os.path.join(ROOT, "vision_amd", "csrc"), str(src), "-o", exe], check=True, capture_output=True)
    rng = random.Random(0)
    bits = [0, 1, 0x7fffff, 0x800000, 0x7f7fffff, 0x7f800000, 0x7fc00000, 0x7fffffff]
    for e in list(range(100, 160)) + [5, 15, 16, 17, 18, 20, 250, 254]:
        for m in (0, 1, 0x5fffff, 0x600000, 0x600001, 0x7dffff, 0x7e0000, 0x7e0001, 0x7fffff, rng.randrange(1 << 23)):
            bits.append(e << 23 | m)
    got = subprocess.run([exe] + [f"{b:x}" for b in bits], check=True, capture_output=True, text=True).stdout.split()
    as_float = lambda b: torch.tensor([b if b < 1 << 31 else b - (1 << 32)], dtype=torch.int32).view(torch.float32).item()
    for b, e4m3, int8 in zip(bits, got[0::2], got[1::2]):
        for text, format in ((e4m3, "e4m3"), (int8, "int8")):
            want, have = kv_plain.power_scale(as_float(b), format), as_float(int(text, 16))
            assert have == want or (math.isnan(have) and math.isnan(want)), (hex(b), format, have, want)


# ---------------------------------------------------------------------------------------------------- the plain forms

def test_plain_code_rounds_like_e4m3():
    x = torch.cat([torch.linspace(-448, 448, 20001), torch.linspace(-0.05, 0.05, 20001), torch.tensor([2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0])])
    assert torch.equal(kv_plain.code(x.double(), "e4m3").float(), x.to(torch.float8_e4m3fn).float())


def test_plain_cache_moves_codes_when_a_scale_grows():
    c = kv_plain.Cache(64, "int8")
    c.append(torch.tensor([[100.0, 1.0]], dtype=torch.float64), 0)
    c.append(torch.tensor([[300.0, -5.0]], dtype=torch.float64), 1)
    assert c.blocks[0][1] == 4.0 and c.read(0, 2, 2).tolist() == [[100.0, 0.0], [300.0, -4.0]]
    c.append(torch.tensor([[1.0, 1.0]], dtype=torch.float64), 0)                  # begins the block anew
    assert c.blocks[0][1] == 2.0 ** -6


# ---------------------------------------------------------------------------------------------------- launches

GRID = r'''
#include "common.h"
using namespace vamd;
int main() {
    const int64_t counts[] = {1, 2, 65535, 65536, kGridFlat - 1, kGridFlat, kGridFlat + 1, 16777215, 16777216, 16777217, 0x40000001, kGridMost};
    for (int64_t n : counts) {
        const dim3 g = grid_of(n);
        if ((uint64_t)g.x * 256 >= 1ull << 32 || g.y > 65535 || g.z != 1) return 1;          // extents in threads, 32 bits each
        if ((int64_t)g.x * g.y < n || (int64_t)g.x * g.y >= n + kGridRow) return 2;
        if (g.y > 1 && g.x != kGridRow) return 3;                                             // what block_number() takes a row to be
    }
    return 0;
}
'''


def test_a_launch_holds_all_its_workgroups(tmp_path):
    src = tmp_path / "grid.hip"
    src.write_text(GRID)
    exe = str(tmp_path / "grid")
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "--offload-host-only", "-O1", "-std=c++17", "-I",
                    os.path.join(ROOT, "vision_amd", "csrc"), str(src), "-o", exe], check=True, capture_output=True)
    assert subprocess.run([exe]).returncode == 0


def test_calls_whose_size_passes_64_bits_are_refused():
    most = 2 ** 31 - 1
    assert rotary_call(batch=most, tokens=most, dim=65536, turned=2, q_heads=65536) < 0 and b"too many" in lib.vamd_last_error()
    for name in ("vamd_kv_append", "vamd_kv_read"):
        assert io_call(name, sequences=most, most=most, rows=most, offsets=P, heads=65536) < 0 and b"too many" in lib.vamd_last_error()


# ---------------------------------------------------------------------------------------------------- what torch has to know

@pytest.fixture
def launches(monkeypatch):
    """Lets calls with CPU tensors pass up to their launch, and collects those instead."""
    made = []
    monkeypatch.setattr(KVCache, "__init__", lambda self, *a, _init=KVCache.__init__, **kw: (_init(self, *a, **kw), setattr(self, "_index", 0))[0])
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    for module in ("vision_amd.kvcache", "vision_amd.rotary"):
        monkeypatch.setattr(module + ".call_on", lambda device, name, *args: made.append((name, args)))
    return made


def test_autograd_notices_what_is_overwritten(launches):
    """A backward pass that has saved a tensor which is then given as `out` refuses to run."""
    def saved(shape):
        w = torch.ones(shape, requires_grad=True)
        out = torch.ones(shape)
        return out, (w * out).sum()
    out, z = saved((2, 6, 32))
    _call("attend", out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    for i in range(2):
        out, z = saved((2, 2, 32))
        other = torch.zeros(2, 2, 32)
        _call("read", out=(out, other) if i == 0 else (other, out))
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.backward()
    assert [name for name, _ in launches] == ["vamd_kv_attend", "vamd_kv_read", "vamd_kv_read"]
    with torch.inference_mode():                            # no version to count there
        _call("attend", out=torch.ones(2, 6, 32))
    assert len(launches) == 4


def test_forward_mode_is_passed_on_or_refused(launches):
    """A dual tensor's tangent is never dropped.  (What Rotary's tangents are: tests/test_rotary_modes_gpu.py.)"""
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        def dual(*shape):
            return forward_ad.make_dual(torch.ones(shape), torch.ones(shape))
        r, pos = Rotary(32), torch.arange(2)
        yq, yk = r(pos, torch.ones(2, 4, 32), dual(2, 1, 32))
        assert forward_ad.unpack_dual(yq).tangent is None and forward_ad.unpack_dual(yk).tangent.shape == yk.shape
        assert len(launches) == 3                           # two tensors, one tangent
        for q, k in ((dual(2, 4, 32), None), (torch.ones(2, 4, 32), dual(2, 1, 32))):
            with pytest.raises(RuntimeError, match="tangent"):
                r.apply_(pos, q, k)
        for method, bad in (("append", lambda: dict(k=dual(2, 2, 32))), ("append", lambda: dict(v=dual(2, 2, 32))), ("attend", lambda: dict(q=dual(2, 6, 32))),
                            ("attend", lambda: dict(out=dual(2, 6, 32))), ("read", lambda: dict(out=(torch.ones(2, 2, 32), dual(2, 2, 32))))):
            with pytest.raises(RuntimeError, match="tangent"):
                _call(method, **bad())
        assert len(launches) == 3
        _call("attend")
    assert len(launches) == 4


def _every_call():
    r, pos = Rotary(32), torch.arange(2)
    yield "forward", lambda q: r(pos, q)
    yield "apply_", lambda q: r.apply_(pos, q)
    c, table, start = KVCache(4, 6, 32, device="cpu"), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    yield "append", lambda q: c.append(q, q, table, start)
    yield "read", lambda q: c.read(table, start, 2, out=(q, torch.zeros(2, 6, 32)))
    yield "attend", lambda q: c.attend(q, table, start)


def _without_a_launch(monkeypatch):
    """As `launches`, but with call_on's own checks."""
    monkeypatch.setattr(KVCache, "__init__", lambda self, *a, _init=KVCache.__init__, **kw: (_init(self, *a, **kw), setattr(self, "_index", 0))[0])
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: None, raising=False)
    made = []
    monkeypatch.setattr(_lib, "_entries", {name: lambda *args, name=name: made.append(name) or 0 for name in _lib.SIGNATURES})
    return made


@pytest.mark.filterwarnings("ignore")
def test_calls_are_not_traced_away(monkeypatch):
    """A recorded program that lacks the launch would return memory that nobody wrote."""
    from torch.fx.experimental.proxy_tensor import make_fx
    made = _without_a_launch(monkeypatch)
    q = torch.ones(2, 6, 32)
    for name, call in _every_call():
        call(q)
        assert len(made) == 1, name
        with pytest.raises(RuntimeError, match="recorded"):
            torch.jit.trace(call, q)
        with pytest.raises(RuntimeError, match="recorded"):
            make_fx(call)(q)
        with pytest.raises(RuntimeError, match="recorded"):
            make_fx(call, pre_dispatch=True)(q)
        for transform in (lambda: torch.func.jvp(call, (q,), (q,)), lambda: torch.func.vmap(call)(q[None]), lambda: make_fx(call, tracing_mode="fake")(q)):
            with pytest.raises(Exception):
                transform()
        assert made.pop() and not made, name


def negated(*shape):
    """A view whose sign torch keeps apart from the memory; features adjacent."""
    t = torch._neg_view(torch.arange(1.0, 1 + math.prod(shape)).view(shape))
    assert t.is_neg() and t.stride(-1) == 1
    return t


def test_lazily_negated_views(launches):
    """Read as what they stand for, not as what lies in memory; not written into."""
    def floats(at, n):
        return [x for x in (ctypes.c_float * n).from_address(at)]
    for name, position, call in (("vamd_rotary", 10, lambda: Rotary(32)(torch.arange(2), negated(2, 6, 32))),
                                 ("vamd_kv_append", 0, lambda: _call("append", k=negated(2, 2, 32))),
                                 ("vamd_kv_append", 3, lambda: _call("append", v=negated(2, 2, 32))),
                                 ("vamd_kv_attend", 0, lambda: _call("attend", q=negated(2, 6, 32)))):
        launches.clear()
        hold = []
        # the launch is where the pointer is valid
        def look(device, entry, *args):
            hold.append((entry, floats(args[position], 3)))
        with pytest.MonkeyPatch.context() as m:
            m.setattr("vision_amd.kvcache.call_on", look)
            m.setattr("vision_amd.rotary.call_on", look)
            call()
        assert hold == [(name, [-1.0, -2.0, -3.0])]
    for call in (lambda: Rotary(32).apply_(torch.arange(2), negated(2, 6, 32)), lambda: _call("attend", out=negated(2, 6, 32)),
                 lambda: _call("read", out=(negated(2, 2, 32), torch.zeros(2, 2, 32)))):
        with pytest.raises(ValueError, match="lazy sign"):
            call()


def test_overlapping_across_storages():
    """Memory that two storages share (another library's buffer, taken over twice)."""
    buf = np.zeros((3, 6, 32), np.float32)
    a, b = torch.from_numpy(buf[:2]), torch.from_numpy(buf[1:])
    assert a.untyped_storage().data_ptr() != b.untyped_storage().data_ptr()
    assert _lib.overlapping(a, b) and _lib.overlapping(b, a) and not _lib.overlapping(a[:1], b)
    with pytest.raises(ValueError, match="share memory"):
        _call("attend", q=a, out=b)
    rng = random.Random(2)
    flat = np.zeros(3000, np.float32)
    for _ in range(300):
        lo, hi = rng.randrange(2000), rng.randrange(2000)
        n, m = rng.randint(1, 900), rng.randint(1, 900)
        x, y = torch.from_numpy(flat[lo:lo + n]), torch.from_numpy(flat[hi:hi + m])
        assert _lib.overlapping(x, y) == (lo < hi + m and hi < lo + n)


def test_a_table_of_one_block_each_has_any_strides(launches):
    table = torch.arange(2, dtype=torch.int32)[None].t()
    assert table.shape == (2, 1) and table.stride() == (1, 2)
    _call("attend", table=table)
    at = launches[0][1].index(table.data_ptr())
    assert launches[0][1][at + 1] == 1                       # rows of the table one entry apart


UNITS = r'''
#include <stdlib.h>
#include "kv_layout.h"
using namespace vamd;
int main() {
    // units are those that spans are found in
    for (int unit = 64; unit <= 256; unit *= 2) for (int start = -2; start < 300; start += 7) for (int n = 0; n < 700; n += 9) {
        int hit = 0;
        for (int j = 0; j < 20; ++j) {
            const KvSpan s = kv_span(start, n, ((start < 0 ? 0 : start) / unit + j) * (int64_t)unit, unit);
            hit += s.hi > s.lo;
        }
        if (hit != kv_units(start, n, unit)) return 1;
    }
    if (kv_units(2147483647, 2147483647, 64) != 33554433) return 2;
    // a batch's units fit into the launch, however its rows lie; without a bound the launch goes by the rows
    srand(1);
    for (int trial = 0; trial < 3000; ++trial) {
        const int B = 1 + rand() % 70, unit = 64 << rand() % 3;
        int64_t rows = 0, units = 0;
        int most = 0;
        for (int b = 0; b < B; ++b) {
            const int n = rand() % 3 ? rand() % 4 : rand() % 3000;
            rows += n;
            most = n > most ? n : most;
            units += kv_units(rand() % 1000, n, unit);
        }
        const KvUnits known = kv_io_units(true, B, rows, most, unit), open = kv_io_units(true, B, rows, (int)rows, unit);
        if (units > known.count || units > open.count) return 3;
        if (open.count > kKvListed * (rows / unit + 2 * B)) return 4;
    }
    const KvUnits u = kv_io_units(true, 256, 1 << 20, 1 << 20, 64), each = kv_io_units(false, 256, 1 << 20, 1 << 12, 64);
    if (!u.listed || u.count != (1 << 14) + 512 || each.listed || each.count != 256 * 65) return 5;
    return 0;
}
'''


def test_units_of_a_batch(tmp_path):
    src = tmp_path / "units.hip"
    src.write_text(UNITS)
    exe = str(tmp_path / "units")
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "--offload-host-only", "-O1", "-std=c++17", "-I",
                    os.path.join(ROOT, "vision_amd", "csrc"), str(src), "-o", exe], check=True, capture_output=True)
    assert subprocess.run([exe]).returncode == 0


PIECES = r'''
#include "kv_layout.h"
using namespace vamd;
int main() {
    for (int D = 16; D <= 256; D += 16) for (int q = 0; q < 4 * D; ++q) {
        int t, d, g;
        kv_key_piece(q, D / 16, t, d);
        for (int f = 0; f < 16; ++f) if (kv_key_at(t, d + f, D) != q * 16 + f) return 1;
        kv_value_piece(q, g, d);
        for (int i = 0; i < 16; ++i) if (kv_value_at(i / 4 * 16 + 4 * g + i % 4, d) != q * 16 + i) return 2;
    }
    // what a lane of the decoding kernel adds to a tile's first piece
    for (int D = 64; D <= 256; D += 64) for (int lane = 0; lane < 64; ++lane) for (int c = 0; c < D / 64; ++c) for (int t = 0; t < 4; ++t)
        if (kv_key_at(t * 16, c * 64, D) + lane * 16 != kv_key_at(t * 16 + (lane & 15), c * 64 + (lane >> 4) * 16, D)) return 3;
    for (int lane = 0; lane < 64; ++lane) for (int s = 0; s < 16; ++s)
        if (kv_value_at(0, s * 16) + lane * 16 != kv_value_at(4 * (lane >> 4), s * 16 + (lane & 15))) return 4;
    return 0;
}
'''


def test_the_layout_both_ways(tmp_path):
    src = tmp_path / "pieces.hip"
    src.write_text(PIECES)
    exe = str(tmp_path / "pieces")
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "--offload-host-only", "-O1", "-std=c++17", "-I",
                    os.path.join(ROOT, "vision_amd", "csrc"), str(src), "-o", exe], check=True, capture_output=True)
    assert subprocess.run([exe]).returncode == 0


def test_rotary_refuses_keys_of_too_few_dimensions():
    r, pos = Rotary(32), torch.tensor(3)
    for k in (torch.zeros(32), torch.zeros(())):             # beside queries [heads, head_dim]
        for call in (r, r.apply_):
            with pytest.raises(ValueError, match="differ"):
                call(pos, torch.zeros(4, 32), k)


def test_a_call_of_rotary_is_one_call_to_its_hooks(launches):
    from torch.autograd import forward_ad
    r, pos, seen = Rotary(32), torch.arange(2), []
    r.register_forward_hook(lambda module, args, out: seen.append(len(args)))
    r(pos, torch.ones(2, 4, 32), torch.ones(2, 0, 32))
    with forward_ad.dual_level():
        r(pos, torch.ones(2, 4, 32), forward_ad.make_dual(torch.ones(2, 1, 32), torch.ones(2, 1, 32)))
    assert seen == [3, 3]
