"""CPU: what the packed attention, the appending page write and the 4-bit cache's calls refuse,
before any launch (no pointer is read here)."""
import ctypes as C
import math

import pytest

from puter_amd import _lib

FAKE = 0x1000
F32, F16, BF16, E4M3, I32, I4 = 0, 1, 2, 3, 5, 7


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def rope(**kw):
    f = dict(base_freq=1e4, start_position=0, mode=1, scaling=0, scaling_factor=1.0, low_freq_factor=0.0,
             high_freq_factor=0.0, original_context=0)
    f.update(kw)
    return _lib.RopeConfig(**f)


APPEND = dict(config="rope", query=FAKE, key=FAKE, value=FAKE, positions=FAKE, ids=FAKE, offsets=FAKE, qout=FAKE,
              kpages=FAKE, vpages=FAKE, kpar=FAKE, vpar=FAKE, rows=4, qh=8, kvh=2, dim=128, qs=1024, ks=256, vs=256,
              pages=4, page_size=16, group=64, dtype=BF16, cache=I4, status=None, stream=None)


def append(lib, **kw):
    a = dict(APPEND, **kw)
    if a["config"] == "rope":
        a["config"] = rope()
    if a["config"] is not None:
        a["config"] = C.byref(a["config"])
    return lib.puter_hip_kv_page_append_rope(*a.values())


@pytest.mark.parametrize("change", [
    dict(dtype=I32), dict(dtype=E4M3), dict(cache=F16), dict(cache=6), dict(dtype=F16, cache=BF16),
    dict(rows=-1), dict(qh=-1), dict(kvh=0), dict(dim=0), dict(pages=-1), dict(page_size=0),
    dict(dim=127, cache=BF16), dict(dim=1026, cache=BF16, qs=9000, ks=9000, vs=9000),
    dict(qs=1023), dict(ks=255), dict(vs=255),
    dict(dim=96), dict(dim=32, group=32), dict(group=16), dict(group=0), dict(group=256), dict(dim=64, group=128),
    dict(kpages=FAKE + 8), dict(vpages=FAKE + 4), dict(kpar=FAKE + 2), dict(vpar=FAKE + 1), dict(status=FAKE + 2),
    dict(config=rope(base_freq=0.0)), dict(config=rope(mode=2)), dict(config=rope(scaling=2)),
    dict(config=rope(scaling=1, scaling_factor=8.0, low_freq_factor=4.0, high_freq_factor=1.0, original_context=8)),
    dict(config=rope(base_freq=math.inf)), dict(config=rope(base_freq=math.nan)), dict(config=rope(start_position=1 << 46)),
    dict(config=rope(start_position=-(1 << 62))), dict(config=rope(base_freq=1e-9)),
    dict(config=rope(scaling=1, scaling_factor=1e-5, low_freq_factor=1.0, high_freq_factor=4.0, original_context=8)),
    dict(qh=70000, qs=70000 * 128), dict(kvh=70000, ks=70000 * 128, vs=70000 * 128),
])
def test_append_refuses(lib, change):
    assert append(lib, **change) == _lib.ERR_INVALID
    assert lib.puter_hip_last_error().startswith(b"kv append")


@pytest.mark.parametrize("name", ["query", "key", "value", "positions", "ids", "offsets", "qout", "kpages", "vpages",
                                  "kpar", "vpar"])
def test_append_nil(lib, name):
    assert append(lib, **{name: None}) == _lib.ERR_NIL


def test_append_nothing_to_do(lib):
    none = dict.fromkeys(["query", "key", "value", "positions", "ids", "offsets", "qout", "kpages", "vpages", "kpar",
                          "vpar"])
    assert append(lib, rows=0, **none) == _lib.OK


GATHER = dict(pages=FAKE, params=FAKE, table=FAKE, out=FAKE, count=4, page_size=16, kvh=2, dim=128, group=64, rows=8,
              dtype=BF16, status=None, stream=None)


def test_gather_refuses(lib):
    def call(**kw):
        return lib.puter_hip_kv_page_gather_int4(*dict(GATHER, **kw).values())
    for change in (dict(dtype=I4), dict(dtype=E4M3), dict(count=-1), dict(page_size=0), dict(page_size=1 << 31), dict(kvh=0), dict(rows=-1), dict(rows=1 << 31),
                   dict(dim=80), dict(group=48), dict(dim=64, group=128), dict(pages=FAKE + 2), dict(params=FAKE + 1),
                   dict(status=FAKE + 3), dict(kvh=70000), dict(rows=1 << 60)):
        assert call(**change) == _lib.ERR_INVALID, change
    for name in ("pages", "params", "table", "out"):
        assert call(**{name: None}) == _lib.ERR_NIL
    assert call(rows=0, pages=None, params=None, table=None, out=None) == _lib.OK


PACKED = dict(q=FAKE, k=FAKE, v=FAKE, o=FAKE, qoff=FAKE, koff=FAKE, batch=2, total_q=8, total_k=8, dtype=BF16,
              status=None, stream=None)


def test_packed_refuses(lib):
    def call(cfg=(8, 64, 1, 0, 0, 0.0, 0, 2), **kw):
        c = C.byref(_lib.MHAConfig(*cfg)) if cfg else None
        return lib.puter_hip_multi_head_attention_packed(c, *dict(PACKED, **kw).values())
    assert call(cfg=None) == _lib.ERR_NIL
    for cfg in ((6, 64, 1, 0, 0, 0.0, 0, 4), (8, 257, 1, 0, 0, 0.0, 0, 2), (0, 64, 1, 0, 0, 0.0, 0, 0),
                (8, 0, 1, 0, 0, 0.0, 0, 2), (8, 64, 1, 0, -1, 0.0, 0, 2), (70000, 64, 1, 0, 0, 0.0, 0, 2)):
        assert call(cfg=cfg) == _lib.ERR_INVALID, cfg
    for change in (dict(dtype=E4M3), dict(batch=-1), dict(total_q=-1), dict(total_k=-1), dict(status=FAKE + 2),
                   dict(total_q=1 << 30), dict(total_k=1 << 30), dict(koff=None, total_k=7)):
        assert call(**change) == _lib.ERR_INVALID, change
    for name in ("q", "k", "v", "o", "qoff"):
        assert call(**{name: None}) == _lib.ERR_NIL
    none = dict.fromkeys(["q", "k", "v", "o", "qoff", "koff"])
    assert call(batch=0, **none) == _lib.OK
    assert call(total_q=0, **none) == _lib.OK


ATTEND = dict(q=FAKE, kp=FAKE, vp=FAKE, kpar=FAKE, vpar=FAKE, table=FAKE, ctx=FAKE, batch=2, query_len=1, max_pages=4,
              page_size=16, num_pages=8, heads=8, kvh=2, dim=128, group=64, max_context=64, dtype=BF16, out=FAKE, ws=FAKE,
              ws_bytes=1 << 30, stream=None)


def attend(lib, **kw):
    return lib.puter_hip_paged_int4_attention(*dict(ATTEND, **kw).values())


@pytest.mark.parametrize("change", [
    dict(dtype=F32), dict(dtype=E4M3), dict(batch=-1), dict(query_len=-1), dict(page_size=0), dict(num_pages=-1),
    dict(heads=0), dict(kvh=0), dict(heads=7), dict(dim=96), dict(dim=80, group=32), dict(group=16),
    dict(dim=64, group=128), dict(max_context=65), dict(max_context=0), dict(ws_bytes=0), dict(batch=70000),
    dict(query_len=70000), dict(num_pages=1 << 28), dict(max_pages=1 << 28), dict(page_size=1 << 32),
    dict(q=FAKE + 8), dict(kp=FAKE + 8), dict(vp=FAKE + 4), dict(kpar=FAKE + 8), dict(vpar=FAKE + 4), dict(out=FAKE + 2),
    dict(ws=FAKE + 8)])
def test_int4_refuses(lib, change):
    assert attend(lib, **change) == _lib.ERR_INVALID
    assert lib.puter_hip_last_error().startswith(b"paged int4")


def test_int4_nil_and_nothing(lib):
    for name in ("q", "kp", "vp", "kpar", "vpar", "table", "ctx", "out", "ws"):
        assert attend(lib, **{name: None}) == _lib.ERR_NIL, name
    none = dict.fromkeys(["q", "kp", "vp", "kpar", "vpar", "table", "ctx", "out", "ws"])
    assert attend(lib, batch=0, **none) == _lib.OK
    assert attend(lib, query_len=0, **none) == _lib.OK
    assert lib.puter_hip_paged_int4_workspace_bytes(0, 1, 8, 2, 128, 64) == 0
