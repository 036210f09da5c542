"""CPU: what the paged key / value cache's entry points refuse, before any launch."""
import ctypes as C

import pytest
import torch


def _cache(**kw):
    from merv_amd import _lib
    base = dict(k_pages=4096, v_pages=8192, k_scales=0, v_scales=0, table=4096, n_pages=4, stride_page=2 * 16 * 64, stride_head=16 * 64, stride_token=64,
                scale_stride_page=32, scale_stride_head=16, table_stride=2, rows=3, table_width=2, kv_heads=2, head_dim=64, page_size=16,
                format=_lib.KV_BF16)
    base.update(kw)
    return _lib.PagedCache(**base)


BAD_CACHES = [(dict(format=2), "format"), (dict(head_dim=96), "head_dim"), (dict(page_size=24), "page_size"), (dict(page_size=8), "page_size"),
              (dict(page_size=2048), "page_size"), (dict(kv_heads=0), "geometry"), (dict(rows=-1), "geometry"), (dict(n_pages=-1), "geometry"),
              (dict(k_pages=0), "null pages"), (dict(table=0), "null table"), (dict(k_pages=4104), "16-byte"), (dict(stride_token=68), "16-byte"),
              (dict(format=1), "scales"), (dict(format=1, k_scales=64, v_scales=66), "4-byte"), (dict(format=1, k_scales=64, v_scales=64, stride_head=1032), "16-byte"),
              (dict(format=1, k_scales=64, v_scales=64, scale_stride_page=30), "4-byte")]


@pytest.mark.parametrize("bad,msg", BAD_CACHES, ids=[str(b) for b, _ in BAD_CACHES])
def test_bad_caches_are_refused(bad, msg):
    from merv_amd import _lib
    lib, cache = _lib.load(), _cache(**bad)
    calls = [lambda: lib.merv_paged_cache_write(cache, 64, 128, 64, 64, 128, 64, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 64, 64, 3, 0, 0),
             lambda: lib.merv_paged_cache_read(cache, 64, 128, 64, 64, 128, 64, 64, 0, 3, 0),
             lambda: lib.merv_paged_decode_attention(cache, 64, 256, 64, 64, 256, 64, 0, 64, 4, 0, 1.0, 4096, 1 << 30, 0)]
    for call in calls:
        with pytest.raises(ValueError, match=msg):
            _lib.check(call(), "paged")


def test_bad_calls_are_refused():
    from merv_amd import _lib
    lib, c = _lib.load(), _cache()

    def write(**kw):
        a = dict(k=64, ks=128, kh=64, v=64, vs=128, vh=64, q=0, qs=0, qh=0, cos=0, sin=0, rl=0, rs=0, qo=0, qos=0, qoh=0, ko=0, kos=0, koh=0, off=64, start=64,
                 T=5, H=0, st=0)
        a.update(kw)
        return lib.merv_paged_cache_write(c, *a.values())

    rope = dict(cos=64, sin=64, rl=10, rs=64)
    for kw, msg in [(dict(k=0), "null"), (dict(start=0), "null"), (dict(T=-1), "geometry"), (dict(off=0), "one token for each row"), (dict(cos=64), "together"),
                    (dict(q=64, qo=64, H=4), "q needs"), (dict(q=64, H=4, **rope), "q needs"), (dict(q=64, qo=64, H=0, **rope), "q needs"),
                    (dict(rope, rl=0), "rotary tables"), (dict(rope, rs=32), "rotary tables"), (dict(rope, cos=72), "rotary tables"), (dict(k=72), "16-byte"),
                    (dict(vs=100), "16-byte"), (dict(ko=64, kos=4), "16-byte")]:
        with pytest.raises(ValueError, match=msg):
            _lib.check(write(**kw), "write")
    for args, msg in [((0, 128, 64, 64, 128, 64, 64, 0, 3, 0), "null"), ((64, 128, 64, 64, 128, 64, 0, 0, 3, 0), "null"),
                      ((64, 128, 64, 64, 128, 64, 64, 0, -1, 0), "geometry"), ((64, 128, 4, 64, 128, 64, 64, 0, 3, 0), "16-byte")]:
        with pytest.raises(ValueError, match=msg):
            _lib.check(lib.merv_paged_cache_read(c, *args), "read")
    for args, msg in [((0, 256, 64, 64, 256, 64, 0, 64, 4, 0, 1.0, 4096, 1 << 30, 0), "null"), ((64, 256, 64, 64, 256, 64, 0, 0, 4, 0, 1.0, 4096, 1 << 30, 0), "null"),
                      ((64, 256, 64, 64, 256, 64, 0, 64, 5, 0, 1.0, 4096, 1 << 30, 0), "multiple"), ((64, 256, 64, 64, 256, 64, 0, 64, 0, 0, 1.0, 4096, 1 << 30, 0), "multiple"),
                      ((64, 250, 64, 64, 256, 64, 0, 64, 4, 0, 1.0, 4096, 1 << 30, 0), "16-byte"), ((72, 256, 64, 64, 256, 64, 0, 64, 4, 0, 1.0, 4096, 1 << 30, 0), "16-byte")]:
        with pytest.raises(ValueError, match=msg):
            _lib.check(lib.merv_paged_decode_attention(c, *args), "attention")
    # calls that a launch could not cover
    big = _cache(rows=1 << 20, kv_heads=1 << 11, n_pages=0, k_pages=0, v_pages=0)
    edge = _cache(rows=1, kv_heads=1, n_pages=0, k_pages=0, v_pages=0)  # 2^32 threads, one more than a launch has
    for rc in (lambda: lib.merv_paged_cache_write(edge, 64, 128, 64, 64, 128, 64, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 64, 64, (1 << 28) - 1, 0, 0),
               lambda: lib.merv_paged_cache_read(edge, 64, 128, 64, 64, 128, 64, 64, 0, (1 << 28) - 1, 0),
               lambda: lib.merv_paged_cache_write(big, 64, 128, 64, 64, 128, 64, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 64, 64, 1 << 18, 0, 0),
               lambda: lib.merv_paged_cache_read(big, 64, 128, 64, 64, 128, 64, 64, 0, 1 << 18, 0),
               lambda: lib.merv_paged_decode_attention(big, 64, 256, 64, 64, 256, 64, 0, 64, 1 << 11, 0, 1.0, 4096, 1 << 30, 0),
               lambda: lib.merv_paged_decode_attention(_cache(table_width=1 << 27), 64, 256, 64, 64, 256, 64, 0, 64, 4, 0, 1.0, 4096, 1 << 30, 0),
               lambda: lib.merv_paged_decode_attention(_cache(table_width=1 << 24, rows=1 << 10), 64, 256, 64, 64, 256, 64, 0, 64, 4, 0, 1.0, 4096, 1 << 30, 0),
               lambda: lib.merv_paged_decode_attention(_cache(stride_token=1 << 26), 64, 256, 64, 64, 256, 64, 0, 64, 4, 0, 1.0, 4096, 1 << 30, 0)):
        with pytest.raises(ValueError, match="at most"):
            _lib.check(rc(), "paged")
    with pytest.raises(ValueError, match="workspace too small"):  # 2048 positions a row, few pairs: shared out, which takes a workspace
        _lib.check(lib.merv_paged_decode_attention(_cache(table_width=128), 64, 256, 64, 64, 256, 64, 0, 64, 4, 0, 1.0, 4096, 100, 0), "attention")
    need = lib.merv_paged_decode_attention_workspace_bytes(3, 4, 2, 64, 2048)
    assert need == 3 * 2 * 16 * (16 + 2 * 2 * 68 * 4) and lib.merv_paged_decode_attention_workspace_bytes(3, 4, 2, 64, 512) == 0
    assert lib.merv_paged_decode_attention_workspace_bytes(3, 5, 2, 64, 2048) == 0
    with pytest.raises(ValueError, match="null"):
        _lib.check(lib.merv_paged_decode_attention(C.POINTER(_lib.PagedCache)(), 64, 256, 64, 64, 256, 64, 0, 64, 4, 0, 1.0, 0, 0, 0), "attention")


def test_tensors_on_the_cpu_are_refused():
    """There is no CPU path: the wrappers say so instead of handing host pointers to a kernel."""
    from merv_amd import ops
    pages = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    table, n = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    k, q = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_cache_write(k, k, pages, pages, table, n)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_cache_read(pages, pages, table, None, torch.zeros(4, dtype=torch.int32), 0)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_decode_attention(q, pages, pages, table, n)


def test_the_packed_structure_is_the_c_one():
    from merv_amd import _lib, ops
    values = [(i + 1) * 16 for i in range(len(_lib.PagedCache._fields_))]
    assert ops._PAGED_CACHE.size == C.sizeof(_lib.PagedCache)
    c = _lib.PagedCache.from_buffer_copy(ops._PAGED_CACHE.pack(*values))
    assert [getattr(c, n) for n, _ in _lib.PagedCache._fields_] == values


PLAN = r"""
#include <vector>
#include "paged_split.h"
using namespace merv;
// 0: every unit of every row's pairs is done once, by a worker that has it in the segment it is said to, into a slot of its own, and the join
// of a pair reads just the slots that were written for it; else a number that names what is wrong
extern "C" int walk(const int* lens, int rows, int pairs, int window, int capacity, int most, int* used) {
    int total = 0;
    std::vector<int> first(rows + 1);
    for (int r = 0; r < rows; ++r) {
        const PagedSpan s = paged_span(lens[r], window, capacity);
        if (lens[r] > 0 && lens[r] <= capacity) {
            if (s.units < 1 || s.base % 16 || s.base > s.lo || s.lo - s.base > 15) return 1;
            if (s.base + s.units * PAGED_UNIT < s.len || s.base + (s.units - 1) * PAGED_UNIT >= s.len) return 2;
            if (s.len - s.lo != (window > 0 && window < lens[r] ? window : lens[r])) return 3;
        } else if (s.units) return 4;
        first[r] = total;
        total += s.units * pairs;
    }
    first[rows] = total;
    const PagedShare sh = paged_share(total, most);
    const int W = *used = sh.workers;
    if (W > 0 && paged_start(sh, W) != total) return 5;
    std::vector<int> done(total), slot_of(total, -1), taken(2 * (most > 0 ? most : 1)), last_of(most > 0 ? most : 1, -1), open_slot(most > 0 ? most : 1, -1);
    for (int w = 0; w < W; ++w) {
        const int a = paged_start(sh, w), b = paged_start(sh, w + 1);
        if (b - a < total / W || b - a > total / W + 1 || b <= a) return 6;
        for (int x = a; x < b;) {
            if (paged_owner(sh, x) != w || paged_owner(sh, b - 1) != w) return 7;
            int r = 0;
            while (first[r + 1] <= x) ++r;
            const int n = paged_span(lens[r], window, capacity).units, u = (x - first[r]) % n;
            const int m = n - u < b - x ? n - u : b - x;
            const int slot = m == n ? -1 : paged_slot(w, x == a);
            if (slot >= 0 && taken[slot]++) return 8;
            if (u == 0 && m < n) {  // the pair goes on in later workers: one such pair at most
                if (last_of[w] >= 0) return 9;
                last_of[w] = paged_owner(sh, x + n - 1);
                open_slot[w] = slot;
            }
            for (int y = x; y < x + m; ++y) done[y]++, slot_of[y] = slot;
            x += m;
        }
    }
    for (int x = 0; x < total; ++x) if (done[x] != 1) return 10;
    int joined = 0, parts = 0;
    for (int w = 0; w < W; ++w) {
        if (last_of[w] < 0) continue;
        if (last_of[w] <= w || last_of[w] >= W) return 11;
        for (int v = w; v <= last_of[w]; ++v) {
            const int slot = v == w ? open_slot[w] : 2 * v;
            if (slot < 0 || taken[slot] != 1) return 12;
            taken[slot] = 2;  // read, once
            ++joined;
        }
    }
    for (int t : taken) parts += t != 0;
    return parts == joined ? 0 : 13;
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    import subprocess
    from pathlib import Path
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(PLAN)
    csrc = Path(__file__).resolve().parent.parent / "merv_amd" / "csrc"
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", f"-I{csrc}", "-o", str(d / "plan.so"), str(d / "plan.cpp")])
    fn = C.CDLL(str(d / "plan.so")).walk
    fn.argtypes = [C.POINTER(C.c_int)] + [C.c_int] * 5 + [C.POINTER(C.c_int)]
    return fn


def test_the_work_is_shared_out_whole(walk):
    """The split of the one-token attention over workgroups (paged_split.h): any lengths (none, too long, negative), windows, heads, worker counts."""
    import random
    rng = random.Random(0)
    cases = [([1], 1, 0, 64, 512), ([131072], 8, 0, 131072, 512), ([0, 0], 4, 0, 64, 512), ([-5, 3, 10**6], 2, 0, 256, 512), ([129], 1, 1, 256, 512)]
    for _ in range(400):
        top = rng.choice([5, 130, 1000, 6000])
        cases.append(([rng.randint(-1, top + 3) for _ in range(rng.randint(1, 40))], rng.randint(1, 9), rng.choice([0, 0, 1, 15, 16, 17, rng.randint(1, top)]), top,
                      rng.choice([1, 2, 3, 7, 64, 512])))
    for lens, pairs, window, capacity, most in cases:
        used = C.c_int(-1)
        rc = walk((C.c_int * len(lens))(*lens), len(lens), pairs, window, capacity, most, C.byref(used))
        assert rc == 0, (rc, lens, pairs, window, capacity, most)
        assert 0 <= used.value <= most


def test_pages_are_handed_out_once():
    from merv_amd.paged import PagedKVCache
    c = PagedKVCache(2, 3, 100, 2, 64, "cpu", "e4m3", page_size=16, n_pages=12)
    table = c.table
    c.assign([100, 0, 17])
    assert c.table is table and table.shape == (3, 7)
    used = table[table >= 0].tolist()
    assert len(used) == len(set(used)) == 9 and max(used) < 12
    assert (table[1] == -1).all() and (table[2, :2] >= 0).all() and (table[2, 2:] == -1).all()
    lay = c.layer(1)
    assert lay["k_pages"].shape == (12, 2, 16, 64) and lay["k_scales"].shape == (12, 2, 16) and lay["table"] is table
    c.assign([0, 16, 0])
    assert (c.table >= 0).sum() == 1
    for bad, msg in (([100, 100, 100], "pages needed"), ([101, 0, 0], "at most"), ([1, 1], "3 rows"), ([-1, 0, 0], "at most")):
        with pytest.raises(ValueError, match=msg):
            c.assign(bad)
    with pytest.raises(ValueError, match="format"):
        PagedKVCache(1, 1, 16, 1, 64, "cpu", "fp4")
    with pytest.raises(ValueError, match="page_size"):
        PagedKVCache(1, 1, 16, 1, 64, "cpu", page_size=24)
