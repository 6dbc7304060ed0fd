"""CPU: the checks of a step's sequences and what the kernels read of them
(sulimo_amd/csrc/seq_plan.h, compiled here), and the refusals of the calls that need no device."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

from sulimo_amd import hip
from tests import step_reference as R

CSRC = os.path.join(os.path.dirname(hip.__file__), "csrc")

SOURCE = r'''
#include "seq_plan.h"
#include <string.h>
using namespace sulimo;
static std::string why;
extern "C" const char *shape_error(size_t h, size_t hk, size_t d, size_t w, size_t p, size_t n) {
  why = check_seq_shape(h, hk, d, w, p, n);
  return why.c_str();
}
// q: what an earlier set left; the blob and the tiles go to out, their sizes to sizes
extern "C" const char *plan(int heads, int page, int pages, size_t n, const uint32_t *nn, const uint32_t *st,
                            const uint32_t *table, size_t width, int32_t *out, size_t *sizes) {
  SeqShape g{heads, 1, 64, 0, page, pages};
  Seqs q;
  q.rows = 77;
  why = plan_seqs(g, n, nn, st, table, width, &q);
  if (!why.empty()) {
    if (q.rows != 77) why = "a refused set changed the batch";
    return why.c_str();
  }
  const SeqBlob b = seq_blob(g, q);
  memcpy(out, b.data.data(), b.data.size() * 4);
  const size_t s[] = {b.start, b.page_off, b.row_seq, b.row_slot, b.pages, b.data.size(), (size_t)q.rows, (size_t)q.positions};
  memcpy(sizes, s, sizeof s);
  int32_t *t = out + b.data.size();
  size_t k = 0;
  for (const LoadTile &l : load_tiles(q)) {
    t[4 * k] = l.page_off; t[4 * k + 1] = l.pos; t[4 * k + 2] = l.out_row; t[4 * k++ + 3] = l.count;
  }
  sizes[8] = k;
  return "";
}
// the pieces of all sequences, 8 numbers each, and their count, counters and record rows
extern "C" void pieces(int heads, int kv_heads, int hd, int window, size_t n, const uint32_t *nn, const uint32_t *st, int rows,
                       int key_tile, int group_heads, int sub, int slots, int32_t *out, size_t *sizes) {
  SeqShape g{heads, kv_heads, hd, window, 0, 0};
  Seqs q;
  plan_seqs(g, n, nn, st, nullptr, 0, &q);
  std::vector<int> all(n);
  for (size_t s = 0; s < n; s++) all[s] = (int)s;
  const AttnPlan p = plan_attention_pieces(g, q, all, AttnSplit{rows, key_tile, group_heads, sub, slots, 256, 5.0, 1.0, 2.0, 1.5, 3.0});
  memcpy(out, p.pieces.data(), p.pieces.size() * sizeof(AttnPiece));
  sizes[0] = p.pieces.size();
  sizes[1] = (size_t)p.counters;
  sizes[2] = p.rec_rows;
}
// the pieces of a step's direct lists
extern "C" void direct(int heads, int kv_heads, int hd, size_t n, const uint32_t *nn, const uint32_t *st, int32_t *out, size_t *sizes) {
  SeqShape g{heads, kv_heads, hd, 0, 0, 0};
  Seqs q;
  plan_seqs(g, n, nn, st, nullptr, 0, &q);
  std::vector<int> few, more;
  for (size_t s = 0; s < n; s++) (q.n_new[s] * (heads / kv_heads) <= 16 ? few : more).push_back((int)s);
  AttnPlan a[3];
  plan_direct(g, q, few, more, 256, a);
  for (int i = 0; i < 3; i++) {
    sizes[i] = a[i].pieces.size();
    memcpy(out, a[i].pieces.data(), sizes[i] * sizeof(AttnPiece));
    out += 8 * sizes[i];
  }
}
extern "C" uint32_t divided(uint32_t p, uint32_t d) {
  const FastDiv f = fast_div(d);
  return (uint32_t)(((uint64_t)p * f.magic) >> f.shift);
}
'''


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ is not installed")
    d = tmp_path_factory.mktemp("seq")
    (d / "s.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", CSRC, str(d / "s.cpp"), "-o",
                    str(d / "s.so")], check=True)
    L = C.CDLL(str(d / "s.so"))
    L.shape_error.restype = L.plan.restype = C.c_char_p
    L.shape_error.argtypes = [C.c_size_t] * 6
    L.pieces.argtypes = [C.c_int] * 4 + [C.c_size_t] + [C.c_void_p] * 2 + [C.c_int] * 5 + [C.c_void_p] * 2
    L.direct.argtypes = [C.c_int] * 3 + [C.c_size_t] + [C.c_void_p] * 4
    L.pieces.restype = None
    L.divided.argtypes, L.divided.restype = [C.c_uint32] * 2, C.c_uint32
    L.plan.argtypes = [C.c_int] * 3 + [C.c_size_t] + [C.c_void_p] * 3 + [C.c_size_t] + [C.c_void_p] * 2
    return L


def plan(lib, n_new, start=None, table=None, page=0, pages=0, heads=4, n=None):
    nn = np.asarray(n_new, np.uint32)
    st = None if start is None else np.asarray(start, np.uint32)
    tb = None if table is None else np.ascontiguousarray(table, np.uint32)
    out, sizes = np.zeros(1 << 20, np.int32), np.zeros(9, np.uint64)
    p = [None if a is None else a.ctypes.data for a in (nn, st, tb)]
    why = lib.plan(heads, page, pages, len(nn) if n is None else n, *p, 0 if tb is None else tb.shape[1], out.ctypes.data,
                   sizes.ctypes.data).decode()
    return why, out, [int(x) for x in sizes]


@pytest.mark.parametrize("page,start,new", [(1, [0, 3, 5], [2, 0, 1]), (7, [13, 0, 6], [1, 20, 1]), (64, [64, 63, 0], [64, 2, 0]),
                                            (256, [1000], [300])])
def test_rows_slots_and_tiles(lib, page, start, new):
    need = [-(-(a + b) // page) for a, b in zip(start, new)]
    pages = sum(need) + 3
    order = np.random.default_rng(page).permutation(pages)
    table = np.full((len(new), max(need) + 1), 4000000000, np.uint32)  # entries behind the last are not read
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = order[at:at + k]
        at += k
    why, out, z = plan(lib, new, start, table, page, pages)
    assert why == ""
    n, rows = len(new), sum(new)
    assert z[6] == rows and z[7] == rows + sum(start)
    off = np.concatenate([[0], np.cumsum(new)])
    assert np.array_equal(out[:n + 1], off) and np.array_equal(out[z[0]:z[0] + n], start)
    assert np.array_equal(out[z[2]:z[2] + rows], np.repeat(np.arange(n), new))
    slots = np.concatenate([R.slots(table[s], page, a, a + b) for s, (a, b) in enumerate(zip(start, new))])
    assert np.array_equal(out[z[3]:z[3] + rows], slots)
    page_off = out[z[1]:z[1] + n]
    for s in range(n):
        assert np.array_equal(out[z[4] + page_off[s]:z[4] + page_off[s] + need[s]], table[s, :need[s]])
    # the load tiles cover every position once, in order, and none passes a sequence's end
    tiles = out[z[5]:z[5] + 4 * z[8]].reshape(-1, 4)
    want = [(page_off[s], p) for s in range(n) for p in range(start[s] + new[s])]
    got = [(t[0], t[1] + i) for t in tiles for i in range(t[3])]
    assert got == want
    assert np.array_equal(tiles[:, 2], np.concatenate([[0], np.cumsum(tiles[:, 3])[:-1]]) if len(tiles) else [])


@pytest.mark.parametrize("args,word", [
    (dict(n_new=[1], start=[7], table=[[0, 8]], page=4, pages=8), "n_pages"),
    (dict(n_new=[1], start=[7], table=[[9, 1]], page=4, pages=8), "n_pages"),
    (dict(n_new=[2], start=[7], table=[[0, 1]], page=4, pages=8), "needs 3 pages"),
    (dict(n_new=[1, 1], start=[0, 0], table=[[3], [3]], page=4, pages=8), "twice"),
    (dict(n_new=[8], start=[0], table=[[3, 3]], page=4, pages=8), "twice"),
    (dict(n_new=[1, 1], start=[4, 0], table=[[3, 1], [3, 0]], page=4, pages=8), "elsewhere"),
    (dict(n_new=[1, 0], start=[0, 3], table=[[3], [3]], page=4, pages=8), "elsewhere"),
    (dict(n_new=[1], table=[[0]], page=0, pages=0), "batch with pages"),
    (dict(n_new=[2**31]), "too long"),
    (dict(n_new=[1], start=[2**32 - 1]), "too long"),
    (dict(n_new=[2**30], heads=24), "too long together"),
    (dict(n_new=[1] * 3, start=[2**30] * 3), "too long together"),
    (dict(n_new=[1], n=65536), "65535"),
])
def test_refused_sequences(lib, args, word):
    why, _, _ = plan(lib, **args)
    assert word in why


def test_pages_that_are_only_read_may_be_shared(lib):
    table = [[5, 0], [5, 1], [5, 2]]
    why, _, _ = plan(lib, [1, 1, 0], [4, 6, 4], table, 4, 6)
    assert why == ""


@pytest.mark.parametrize("shape,word", [
    ((12, 5, 128, 0, 0, 0), "multiple"), ((12, 0, 128, 0, 0, 0), "multiple"), ((0, 2, 128, 0, 0, 0), "multiple"),
    ((2048, 2, 128, 0, 0, 0), "multiple"), ((12, 2, 96, 0, 0, 0), "64 or 128"), ((12, 2, 0, 0, 0, 0), "64 or 128"),
    ((0, 0, 0, 5, 0, 0), "head layout"), ((0, 0, 0, 0, 16, 4), "head layout"), ((12, 2, 128, 0, 16, 0), "together"),
    ((12, 2, 128, 0, 0, 4), "together"), ((12, 2, 128, 0, 1 << 16, 1 << 15), "2^31"), ((12, 2, 128, 1 << 31, 0, 0), "window"),
    ((12, 2, 128, 0, 1 << 40, 1 << 40), "2^31"),
])
def test_refused_shapes(lib, shape, word):
    assert word in lib.shape_error(*shape).decode()
    h = C.c_void_p()
    assert hip.lib().sulimo_hip_seq_batch_create(None, *shape, C.byref(h)) == hip.ERR_INVALID_ARGUMENT
    assert word in hip.lib().sulimo_hip_last_error().decode() and not h


def test_calls_without_a_batch_are_refused():
    L = hip.lib()
    h = C.c_void_p()
    assert L.sulimo_hip_seq_batch_create(None, 12, 2, 128, 0, 0, 0, C.byref(h)) == hip.ERR_INVALID_ARGUMENT
    assert L.sulimo_hip_seq_batch_create(None, 12, 2, 128, 0, 0, 0, None) == hip.ERR_INVALID_ARGUMENT
    assert L.sulimo_hip_seq_batch_set(None, 0, None, None, None, 0) == hip.ERR_INVALID_ARGUMENT
    assert L.sulimo_hip_seq_batch_release(None) == hip.OK
    assert L.sulimo_hip_enqueue_kv_store_paged(*[None] * 8) == hip.ERR_INVALID_ARGUMENT
    for f in (L.sulimo_hip_enqueue_kv_load_paged, L.sulimo_hip_enqueue_attention_paged, L.sulimo_hip_enqueue_attention_packed):
        assert f(*[None] * 6) == hip.ERR_INVALID_ARGUMENT
    assert L.sulimo_hip_enqueue_verify_drafts(*[None] * 6, 10, 1.0, None, None) == hip.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("bad", [[-1], [2**32], [1.5], [[1]]])
def test_lengths_that_are_no_lengths_raise(bad):
    with pytest.raises(ValueError):
        hip._u32(bad, (1,))


@pytest.mark.parametrize("rows,key_tile,heads,sub", [(16, 32, 8, 1), (32, 32, 2, 4), (16, 64, 1, 8), (128, 64, 1, 1)])
@pytest.mark.parametrize("slots", [1, 40, 256, 512])
@pytest.mark.parametrize("window", [0, 1, 100])
@pytest.mark.parametrize("new,start", [([1], [0]), ([1], [5000]), ([1, 0, 7, 200], [3, 9, 4000, 70]), ([1] * 300, list(range(300))),
                                       ([2000, 31], [0, 1])])
def test_pieces_cover_every_key_once(lib, rows, key_tile, heads, sub, slots, window, new, start):
    H, Hk = 24, 8
    G = H // Hk
    nn, st = np.asarray(new, np.uint32), np.asarray(start, np.uint32)
    out, z = np.zeros(1 << 18, np.int32), np.zeros(3, np.uint64)
    lib.pieces(H, Hk, 128, window, len(new), nn.ctypes.data, st.ctypes.data, rows, key_tile, heads, sub, slots, out.ctypes.data,
               z.ctypes.data)
    n, counters, rec_rows = (int(x) for x in z)
    p = out[:8 * n].reshape(n, 8)
    assert np.all(np.diff(p[:, 3] - p[:, 2]) <= 0)  # longest first
    tiles = {}
    for seq, row0, t0, t1, piece, np_, rec, counter in p:
        assert t0 < t1
        tiles.setdefault((seq, row0), []).append((piece, t0, t1, np_, rec, counter))
    want = {(s, r) for s in range(len(new)) for r in range(0, new[s] * G, rows)}
    assert set(tiles) == want
    used, recs = set(), []
    for (s, r0), ps in tiles.items():
        ps.sort()
        live = min(rows, new[s] * G - r0)
        first, last = start[s] + r0 // G, start[s] + (r0 + live - 1) // G
        lo = max(0, first - window + 1) if window else 0
        assert [x[0] for x in ps] == list(range(ps[0][3])) and all(x[3:] == ps[0][3:] for x in ps)
        assert ps[0][1] == lo // key_tile and ps[-1][2] == last // key_tile + 1
        assert all(a[2] == b[1] for a, b in zip(ps, ps[1:]))
        if len(ps) > 1:
            groups = Hk // heads
            mine = set(range(ps[0][5], ps[0][5] + groups))
            assert not mine & used and max(mine) < counters
            used |= mine
            recs.append((ps[0][4], ps[0][4] + len(ps) * Hk * live))
    recs.sort()
    assert all(a[1] <= b[0] for a, b in zip(recs, recs[1:])) and (not recs or recs[-1][1] <= rec_rows)


@pytest.mark.parametrize("new,start", [([1], [0]), ([1] * 64, [2000] * 64), ([8], [1000]), ([6] * 64, [2000] * 64),
                                       ([1, 8] * 9, [500] * 18), ([5, 6] * 20, [4000] * 40), ([42, 1, 1], [9000, 10, 3]), ([], [])])
@pytest.mark.parametrize("heads,kv_heads,hd", [(24, 8, 128), (4, 2, 64), (5, 1, 128)])
def test_direct_lists_cover_every_row_once(lib, heads, kv_heads, hd, new, start):
    nn, st = np.asarray(new, np.uint32), np.asarray(start, np.uint32)
    out, z = np.zeros(1 << 18, np.int32), np.zeros(3, np.uint64)
    lib.direct(heads, kv_heads, hd, len(new), nn.ctypes.data, st.ctypes.data, out.ctypes.data, z.ctypes.data)
    p, G, at, seen = out.reshape(-1, 8), heads // kv_heads, 0, set()
    for rows, n in zip((16, 32, 0), (int(x) for x in z)):
        tiles = {(int(seq), int(row0)) for seq, row0, *_ in p[at:at + n]}
        at += n
        assert rows or not n
        for s in {t[0] for t in tiles}:
            assert s not in seen and {t[1] for t in tiles if t[0] == s} == set(range(0, new[s] * G, rows))
        seen |= {t[0] for t in tiles}
    assert seen == set(range(len(new)))


def test_division_by_the_page_size(lib):
    rng = np.random.default_rng(0)
    for d in [1, 2, 3, 5, 7, 16, 48, 64, 100, 255, 256, 1000, 65535, 65536, 10**6 + 3, 2**30, 2**31 - 1]:
        for p in [0, 1, d - 1, d, d + 1, 2 * d - 1, 2 * d, 2**31 - 1, 2**31 - 2] + [int(x) for x in rng.integers(0, 2**31, 200)]:
            if p < 2**31:
                assert lib.divided(p, d) == p // d, (p, d)
