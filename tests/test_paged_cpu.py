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
