"""Rotary positions, the paged key-value cache and paged attention without a GPU: frequencies, descriptor layouts, the
refusals of the C entries (they look at the descriptor before the context), and the address arithmetic of the kernels
compiled for the host."""
import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest

from tests import decode_reference as ref
from torch_engine_b200 import lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts_match_the_header(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text("""
#include <stdio.h>
#include <stddef.h>
#include "te_b200.h"
int main(void) {
    printf("%zu %zu\\n", sizeof(te_rotary_desc), offsetof(te_rotary_desc, reserved));
    printf("%zu %zu\\n", sizeof(te_kv_cache), offsetof(te_kv_cache, reserved));
    printf("%zu %zu\\n", sizeof(te_kv_desc), offsetof(te_kv_desc, position_strides));
    printf("%zu %zu\\n", sizeof(te_paged_attn_desc), offsetof(te_paged_attn_desc, reserved));
    return 0;
}
""")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    rows = [tuple(int(v) for v in line.split()) for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines()]
    mirrors = [(L.RotaryDesc, "reserved"), (L.KvCacheDesc, "reserved"), (L.KvDesc, "position_strides"), (L.PagedAttnDesc, "reserved")]
    assert rows == [(C.sizeof(m), getattr(m, f).offset) for m, f in mirrors]


def test_packed_descriptors_are_the_structures():
    """The struct.pack forms put every field where the ctypes mirrors (and so the header) have it."""
    def fill(desc, start):
        values, n = [], start
        for name, kind in desc._fields_:
            if issubclass(kind, C.Structure):
                inner, n = fill(getattr(desc, name), n)
                values += inner
            elif issubclass(kind, C.Array):
                setattr(desc, name, kind(*range(n, n + kind._length_)))
                values += range(n, n + kind._length_)
                n += kind._length_
            else:
                setattr(desc, name, n)
                values.append(n)
                n += 1
        return values, n
    cache_values = fill(L.KvCacheDesc(), 1)[0]
    for desc, pack in ((L.RotaryDesc(), L.ROTARY_PACK), (L.KvCacheDesc(), L.KV_CACHE_PACK)):
        assert pack.pack(*fill(desc, 1)[0]) == bytes(desc)
    for desc, pack in ((L.KvDesc(), L.KV_PACK), (L.PagedAttnDesc(), L.PAGED_ATTN_PACK)):
        values = fill(desc, 1)[0]
        n = len(cache_values)
        assert L.KV_CACHE_PACK.pack(*values[:n]) + pack.pack(*values[n:]) == bytes(desc)


@pytest.mark.parametrize("rot,base", [(0, 10000.0), (2, 10000.0), (64, 10000.0), (128, 500000.0), (34, 100.0)])
def test_frequencies(rot, base):
    """Against the formulas in Python floats: pow and the few products of either side are within some ulps of 2^-53."""
    j = np.arange(rot // 2)
    plain = base ** (-2.0 * j / max(rot, 1))
    tol = dict(rtol=1e-14, atol=0)
    np.testing.assert_allclose(L.rotary_inv_freq(rot, base), plain, **tol)
    np.testing.assert_allclose(L.rotary_inv_freq(rot, base, L.TE_ROTARY_LINEAR, 4.0), plain / 4, **tol)
    if rot > 2:
        wide = L.rotary_inv_freq(rot, base, L.TE_ROTARY_BASE, 8.0)
        assert wide[0] == 1.0
        np.testing.assert_allclose(wide[-1], plain[-1] / 8, rtol=1e-13)       # the slowest pair is stretched by the factor
    parts = L.rotary_inv_freq(rot, base, L.TE_ROTARY_PARTS, 16.0, 2048, 1.0, 32.0)
    turns = 2048 * plain / (2 * math.pi)
    keep = np.clip((turns - 1.0) / 31.0, 0.0, 1.0)
    np.testing.assert_allclose(parts, plain * (keep + (1 - keep) / 16.0), **tol)


@pytest.mark.parametrize("args", [(-2, 10000.0), (3, 10000.0), (64, 0.0), (64, float("nan")), (64, 1e4, 9), (64, 1e4, L.TE_ROTARY_LINEAR, 0.0),
                                  (2, 1e4, L.TE_ROTARY_BASE, 2.0), (64, 1e4, L.TE_ROTARY_PARTS, 2.0, 0), (64, 1e4, L.TE_ROTARY_PARTS, 2.0, 99, 2.0, 2.0)])
def test_frequencies_refuse(args):
    with pytest.raises(L.BackendError) as e:
        L.rotary_inv_freq(*args)
    assert e.value.status == L.TE_ERR_BAD_ARGUMENT


def _set(desc, **kw):
    for name, value in kw.items():
        at = desc
        *path, last = name.split("__")
        for p in path:
            at = getattr(at, p)
        if isinstance(value, tuple):
            value = type(getattr(at, last))(*value)
        setattr(at, last, value)
    return desc


def rotary_desc(**kw):
    d = L.RotaryDesc()
    d.B, d.H, d.T, d.d, d.rot = 2, 3, 5, 64, 32
    d.x, d.y, d.positions, d.inv_freq, d.scale = 0x1000, 0x9000, 0x2000, 0x3000, 1.0
    return _set(d, **dict(dict(x_strides=(960, 64, 192), y_strides=(960, 320, 64), position_strides=(5, 1)), **kw))


def cache_fields(dtype=L.TE_KV_BF16, prefix="cache__"):
    f = dict(pages=7, heads=2, page_size=16, d=64, k=0x10000, v=0x20000, k_strides=(2048, 1024, 64), v_strides=(2048, 1024, 64), dtype=dtype)
    if dtype == L.TE_KV_E4M3:
        f.update(k_scale=0x5000, v_scale=0x6000, scale_strides=(32, 16, 1))
    return {prefix + k: v for k, v in f.items()}


def kv_desc(dtype=L.TE_KV_BF16, **kw):
    d = _set(L.KvDesc(), **cache_fields(dtype))
    d.B, d.T = 2, 5
    d.k, d.v, d.page_table, d.page_table_stride, d.max_pages, d.positions = 0x1000, 0x2000, 0x3000, 4, 4, 0x4000
    return _set(d, **dict(dict(k_strides=(640, 320, 64), v_strides=(640, 320, 64), position_strides=(5, 1)), **kw))


def attn_desc(dtype=L.TE_KV_BF16, **kw):
    d = _set(L.PagedAttnDesc(), **cache_fields(dtype))
    d.rows, d.q_heads, d.q, d.o, d.page_table, d.page_table_stride, d.max_pages, d.lens = 3, 4, 0x1000, 0x2000, 0x3000, 4, 4, 0x4000
    d.window, d.scale = 0, 0.125
    return _set(d, **dict(dict(q_strides=(256, 64), o_strides=(256, 64)), **kw))


BAD, LAYOUT = L.TE_ERR_BAD_ARGUMENT, L.TE_ERR_UNSUPPORTED_LAYOUT


def answer(entry, d):
    lib = L.load()
    return getattr(lib, entry)(None, C.byref(d), None), lib.te_b200_last_error().decode()


@pytest.mark.parametrize("entry,d", [("te_b200_rotary", rotary_desc()), ("te_b200_kv_append", kv_desc()), ("te_b200_kv_read", kv_desc(L.TE_KV_E4M3)),
                                     ("te_b200_kv_read", kv_desc(k=None)), ("te_b200_paged_attention", attn_desc()),
                                     ("te_b200_rotary", rotary_desc(x=0x9000, x_strides=(960, 320, 64)))])
def test_sound_descriptors_reach_the_context(entry, d):
    assert answer(entry, d) == (BAD, "ctx is NULL")


@pytest.mark.parametrize("kw,code,text", [
    (dict(B=-1), BAD, "bad extents"), (dict(rot=31), BAD, "even"), (dict(rot=66), BAD, "at most d"), (dict(d=1026, rot=4), BAD, "1024"),
    (dict(T=1 << 31), BAD, "2^31"), (dict(B=1 << 20, T=1 << 20), BAD, "2^31"), (dict(x=None), BAD, "NULL"), (dict(y=None), BAD, "NULL"),
    (dict(positions=None), BAD, "NULL"), (dict(inv_freq=None), BAD, "NULL"), (dict(x_strides=(960, -64, 192)), BAD, "negative stride"),
    (dict(y_strides=(960, 0, 64)), LAYOUT, "overlap"), (dict(x=0x9000), LAYOUT, "in place"), (dict(position_strides=(-5, 1)), BAD, "negative stride")])
def test_rotary_refuses(kw, code, text):
    rc, msg = answer("te_b200_rotary", rotary_desc(**kw))
    assert rc == code and text in msg, (rc, msg)


CACHE_REFUSALS = [
    (dict(cache__dtype=3), BAD, "dtype"), (dict(cache__pages=-1), BAD, "extents"), (dict(cache__page_size=0), BAD, "page_size"),
    (dict(cache__page_size=1 << 31), BAD, "page_size"), (dict(cache__d=8), BAD, "multiple of 16"), (dict(cache__d=72), BAD, "multiple of 16"),
    (dict(cache__d=272), BAD, "multiple of 16"), (dict(cache__k=None), BAD, "NULL"), (dict(cache__k=0x10004), LAYOUT, "aligned"),
    (dict(cache__k_strides=(2048, 1024, 60)), LAYOUT, "16 bytes"), (dict(cache__v_strides=(2048, -1024, 64)), BAD, "negative"),
    (dict(cache__page_size=1 << 30, max_pages=2), BAD, "2^31-1"), (dict(cache__heads=1 << 16), BAD, "heads"),
    (dict(max_pages=-1), BAD, "extents"), (dict(page_table=None), BAD, "NULL"), (dict(page_table_stride=-1), BAD, "negative")]


@pytest.mark.parametrize("kw,code,text", CACHE_REFUSALS + [
    (dict(B=-1), BAD, "extents"), (dict(positions=None), BAD, "NULL"), (dict(k_strides=(640, 320, -64)), BAD, "negative"),
    (dict(B=1 << 31), BAD, "2^31"), (dict(B=1 << 30, T=1 << 30), BAD, "too many rows")])
def test_cache_moves_refuse(kw, code, text):
    for entry in ("te_b200_kv_append", "te_b200_kv_read"):
        rc, msg = answer(entry, kv_desc(**kw))
        assert rc == code and text in msg, (entry, rc, msg)


def test_cache_moves_refuse_by_direction():
    assert answer("te_b200_kv_append", kv_desc(k=None))[0] == BAD            # append needs both
    assert answer("te_b200_kv_read", kv_desc(k=None, v=None))[0] == BAD      # read at least one
    assert answer("te_b200_kv_read", kv_desc(k_strides=(640, 0, 64)))[0] == LAYOUT
    assert answer("te_b200_kv_append", kv_desc(k_strides=(640, 0, 64))) == (BAD, "ctx is NULL")      # a broadcast input is read
    assert "scales" in answer("te_b200_kv_append", kv_desc(L.TE_KV_E4M3, cache__k_scale=None))[1]


@pytest.mark.parametrize("kw,code,text", CACHE_REFUSALS + [
    (dict(rows=-1), BAD, "extents"), (dict(q_heads=3), BAD, "multiple"), (dict(cache__heads=0), BAD, "multiple"), (dict(window=-1), BAD, "window"),
    (dict(scale=float("inf")), BAD, "finite"), (dict(q=None), BAD, "NULL"), (dict(o=None), BAD, "NULL"), (dict(lens=None), BAD, "NULL"),
    (dict(o_strides=(256, 32)), LAYOUT, "overlap"), (dict(max_pages=(1 << 27) - 300, q_heads=64), BAD, "too many heads"), (dict(q_strides=(256, -64)), BAD, "negative"), (dict(rows=1 << 31), BAD, "too many")])
def test_paged_attention_refuses(kw, code, text):
    d = attn_desc(**kw)
    n = C.c_size_t()
    rc, msg = answer("te_b200_paged_attention", d)
    assert rc == code and text in msg, (rc, msg)
    assert L.load().te_b200_paged_attention_workspace_size(C.byref(d), 148, C.byref(n)) == code


def test_null_descriptors():
    lib = L.load()
    for entry in ("te_b200_rotary", "te_b200_kv_append", "te_b200_kv_read", "te_b200_paged_attention"):
        assert getattr(lib, entry)(None, None, None) == BAD


def test_places_on_the_host(tmp_path):
    """The division, and page and slot of a position, as the kernels compute them, over page sizes and positions at the
    borders: beyond the table, pages outside the cache, the largest position."""
    src = tmp_path / "places.cpp"
    src.write_text(r"""
#include <stdio.h>
#include <vector>
#include "kv_place.h"
using namespace te;
int main() {
    const uint32_t sizes[] = {1, 2, 3, 5, 7, 13, 16, 31, 33, 64, 100, 127, 1000, 65535, 65536, 65537, 1000003, 0x3fffffffu, 0x40000000u, 0x40000001u, 0x7fffffffu};
    long bad = 0;
    for (uint32_t d : sizes) {
        const FastDivisor f = make_fast_divisor(d);
        uint64_t x = 88172645463325252ull;
        for (int i = 0; i < 200000; ++i) {
            x ^= x << 13; x ^= x >> 7; x ^= x << 17;
            const uint32_t n = (uint32_t)(x >> 33);
            bad += fast_quotient(n, f) != n / d;
            const uint32_t m = n / d * d;                       // a multiple, and its neighbours
            bad += fast_quotient(m, f) != m / d;
            if (m) bad += fast_quotient(m - 1, f) != (m - 1) / d;
        }
        bad += fast_quotient(0x7fffffffu, f) != 0x7fffffffu / d;
        bad += fast_quotient(0, f) != 0;
    }
    const int64_t table[4] = {5, -1, 0, 6};
    const PageRow row = {table, 4, 6};
    const FastDivisor f = make_fast_divisor(13);
    for (int64_t p = -3; p < 60; ++p) {
        int64_t page = -7; uint32_t slot = 0;
        const bool there = kv_place(row, f, p, page, slot);
        const bool want = p >= 0 && p < 52 && table[p / 13] >= 0 && table[p / 13] < 6;
        bad += there != want;
        if (there) bad += page != table[p / 13] || slot != p % 13;
    }
    int64_t page; uint32_t slot;
    bad += kv_place(row, f, INT64_MAX, page, slot) || kv_place(row, f, INT64_MIN, page, slot);
    const PageRow none = {nullptr, 0, 6};
    bad += kv_place(none, f, 0, page, slot);
    printf("%ld\n", bad);
    return 0;
}
""")
    exe = tmp_path / "places"
    subprocess.run(["g++", "-std=c++17", "-O2", "-I", os.path.join(ROOT, "torch-engine_b200", "csrc"), str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.strip() == "0"


def test_eight_bit_grid_of_the_reference():
    """The oracle itself: values on the grid stay, ties go to even, 448 is the top, a row above it takes the next power of two."""
    row = np.array([448.0, 1.0, 0.0625, 17.0, 19.0, -2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10])
    out, unit = ref.e4m3_row(row)
    assert unit == 1.0
    assert out.tolist() == [448.0, 1.0, 0.0625, 16.0, 20.0, -2.0 ** -9, 0.0, 2.0 ** -8]
    assert ref.e4m3_row(np.array([448.0 * (1 + 2.0 ** -20)]))[1] == 2.0
    assert ref.e4m3_row(np.array([0.0]))[1] == 2.0 ** -126


def test_shares_of_paged_attention_on_the_host(tmp_path):
    """Going through all workers' pieces covers every tile of every segment once and in order, the parts of a segment lie in
    the places that the join adds up, and no place is used twice."""
    src = tmp_path / "shares.cpp"
    src.write_text(r"""
#include <stdio.h>
#include <algorithm>
#include <map>
#include <utility>
#include <vector>
#include "paged_plan.h"
using namespace te;
int main() {
    long bad = 0;
    uint64_t x = 88172645463325252ull;
    auto rnd = [&](uint64_t n) { x ^= x << 13; x ^= x >> 7; x ^= x << 17; return x % n; };
    for (int trial = 0; trial < 4000; ++trial) {
        const int tile = trial % 2 ? 64 : 32, heads = 1 + (int)rnd(9), rows = 1 + (int)rnd(12), grid = 1 + (int)rnd(trial % 3 ? 300 : 7);
        const int64_t window = rnd(3) ? 0 : 1 + (int64_t)rnd(500);
        const int most = 3000;
        std::vector<int64_t> len(rows);
        std::vector<int> row_begin(rows + 1, 0);
        for (int r = 0; r < rows; ++r) {
            len[r] = (int64_t)rnd(8) == 0 ? -(int64_t)rnd(3) : (int64_t)rnd(trial % 5 ? 3500 : 70);
            const RowRange range = row_range(len[r], most, window);
            bad += range.n != std::max<int64_t>(0, std::min<int64_t>(len[r], most)) || range.first != (window ? std::max<int64_t>(0, range.n - window) : 0);
            const int c = row_tiles(range, tile);
            if (range.n > range.first) bad += c != (range.n - 1) / tile - range.first / tile + 1; else bad += c != 0;
            row_begin[r + 1] = row_begin[r] + segment_units(c) * heads;
        }
        const int units = row_begin[rows];
        if (!units) continue;
        auto range_of = [&](int r) { return row_range(len[r], most, window); };
        const int workers = std::min(grid, units);
        const Shares shares = shares_of(units, workers);
        bad += share_begin(shares, 0) != 0 || share_begin(shares, workers) != units;
        std::map<std::pair<int, int>, int> done;                            // (row, head tile) -> tiles covered so far
        std::map<int, std::pair<int, int>> place;                           // part slot -> its segment
        std::map<std::pair<int, int>, std::vector<int>> parts;              // segment -> slots in order of its tiles
        std::map<std::pair<int, int>, std::pair<int, int>> join;            // segment -> first and last worker
        for (int w = 0; w < workers; ++w) {
            const int u0 = share_begin(shares, w), u1 = share_begin(shares, w + 1);
            bad += u1 <= u0 || u1 - u0 > units / workers + 1 || worker_of(shares, u0) != w || worker_of(shares, u1 - 1) != w;
            int r = 0;
            while (row_begin[r + 1] <= u0) ++r;
            Walker walk;
            walk.start(u0, u1, r, row_begin[r]);
            Piece p;
            int last_row = -1, last_head = -1;
            while (walk.next(range_of, heads, tile, p)) {
                const std::pair<int, int> seg(p.row, p.head_tile);
                const RowRange range = range_of(p.row);
                const int tiles = row_tiles(range, tile);
                bad += p.row < 0 || p.row >= rows || p.head_tile < 0 || p.head_tile >= heads || p.tiles < 1 || p.range.n != range.n || p.range.first != range.first;
                bad += p.first_tile != range.first / tile + done[seg];          // in order, without gaps
                bad += p.begins != (done[seg] == 0);
                done[seg] += p.tiles;
                bad += p.ends != (done[seg] == tiles) || done[seg] > tiles;
                bad += p.segment_end != row_begin[p.row] + (p.head_tile + 1) * segment_units(tiles);
                bad += p.row < last_row || (p.row == last_row && p.head_tile <= last_head);
                last_row = p.row; last_head = p.head_tile;
                if (!(p.begins && p.ends)) {
                    const int slot = part_slot(w, p.begins);
                    bad += place.count(slot) || slot < 0 || slot >= 2 * workers;
                    place[slot] = seg;
                    parts[seg].push_back(slot);
                }
                if (p.begins && !p.ends) join[seg] = std::make_pair(w, worker_of(shares, p.segment_end - 1));
            }
        }
        for (int r = 0; r < rows; ++r)
            for (int h = 0; h < heads; ++h) {
                const int tiles = row_tiles(range_of(r), tile);
                const std::pair<int, int> seg(r, h);
                bad += done[seg] != tiles;
                if (!parts.count(seg)) { bad += join.count(seg); continue; }
                const std::pair<int, int> j = join.at(seg);
                std::vector<int> want;
                for (int w = j.first; w <= j.second; ++w) want.push_back(part_slot(w, w == j.first));
                bad += want != parts[seg];
            }
    }
    printf("%ld\n", bad);
    return 0;
}
""")
    exe = tmp_path / "shares"
    subprocess.run(["g++", "-std=c++17", "-O2", "-I", os.path.join(ROOT, "torch-engine_b200", "csrc"), str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.strip() == "0"
