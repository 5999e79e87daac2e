"""Host side of laplacesscissors_b200/cache.py: its refusals and the library's.  No GPU: they come before
anything is launched."""
import ctypes as C

import pytest
import torch

import cache_reference as ref
from laplacesscissors_b200 import LsxError, cache
from laplacesscissors_b200._lib import CachePool, CacheRows, CacheView, lib


class HostGpu:
    """Where CPU tensors say they are (get_device), with no context: a call that passes the checks is refused
    by the library, which needs one."""
    device = -1
    handle = C.c_void_p(None)


@pytest.fixture
def host(monkeypatch):
    monkeypatch.setattr(cache, "_stream", lambda device: 0)
    return HostGpu()


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def held(pages=3, heads=2, size=32, D=64, rows=4, width=5):
    return (torch.zeros(cache.pages_shape(pages, heads, size, D), dtype=torch.uint8), ints(rows, width), ints(rows))


def test_layout_covers_each_byte_once():
    for D in (64, 128, 192, 256):
        ref.cell_index(D)
    assert lib.lsx_cache_page_bytes(8, 64, 128) == 8 * 4 * 18 * 128


def test_shapes_are_refused(host):
    pages, tables, lengths = held()
    x = torch.zeros(4, 2, 64)
    for bad in ((64, 3, 63), (64, 8, 64), (64, 0, 64), (64, 40, 128), (1, 32, 320)):
        with pytest.raises(ValueError):
            cache.pages_shape(bad[0], 1, bad[1], bad[2])
    calls = [
        lambda: cache.append(host, x[:, :1], x[:, :1], pages, tables, lengths),
        lambda: cache.append(host, x, x[:3], pages, tables, lengths),
        lambda: cache.append(host, x, x.half(), pages, tables, lengths),
        lambda: cache.append(host, x.double(), x.double(), pages, tables, lengths),
        lambda: cache.append(host, x, x, pages.float(), tables, lengths),
        lambda: cache.append(host, x, x, pages[:, :, :, :63], tables, lengths),
        lambda: cache.append(host, x, x, pages[::2], tables, lengths),
        lambda: cache.append(host, x, x, pages, tables.long(), lengths),
        lambda: cache.append(host, x, x, pages, tables, lengths[:3]),
        lambda: cache.append(host, x[:3], x[:3], pages, tables, lengths, ints(4), sequences=ints(4)),
        lambda: cache.append(host, x[:3], x[:3], pages, tables, lengths, sequences=ints(4)),
        lambda: cache.append(host, torch.zeros(5, 2, 64), torch.zeros(5, 2, 64), pages, tables, lengths),
        lambda: cache.append(host, x.transpose(1, 2), x.transpose(1, 2), pages, tables, lengths),
        lambda: cache.attention(host, torch.zeros(4, 3, 64), pages, tables, lengths),
        lambda: cache.attention(host, torch.zeros(4, 0, 64), pages, tables, lengths),
        lambda: cache.attention(host, torch.zeros(4, 2, 128), pages, tables, lengths),
        lambda: cache.attention(host, x, pages, tables, lengths, out=torch.zeros(4, 2, 64).half()),
        lambda: cache.attention(host, x, pages, tables, lengths, out=torch.zeros(1, 2, 64).expand(4, 2, 64)),
        lambda: cache.attention(host, x, pages, tables, lengths, out=torch.zeros(4, 1, 64).expand(4, 2, 64)),
        lambda: cache.attention(host, x, pages, tables, lengths, torch.zeros(5)),
        lambda: cache.read(host, pages, tables, lengths, ints(5)),
        lambda: cache.read(host, pages, tables, lengths, out=(x, x[:, :, ::2])),
        lambda: cache.read(host, pages, tables, lengths, dtype=torch.float64),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i}")


def test_tensors_that_require_grad_are_refused(host):
    x = torch.zeros(4, 2, 64, requires_grad=True)
    for call in (lambda: cache.append(host, x, x, *held()), lambda: cache.attention(host, x, *held())):
        with pytest.raises(ValueError, match="detach"):
            call()
        with torch.no_grad(), pytest.raises(LsxError, match="context|workspace"):
            call()


def test_page_calls_are_refused(host):
    pool, tables, lengths, refs, listed = torch.zeros(2, 3, 16), ints(4, 5), ints(4), ints(3), ints(2)
    state = (tables, lengths, refs)
    calls = [
        lambda: cache.reserve(host, *state, listed, ints(3), 16),
        lambda: cache.reserve(host, *state, ints(1025), ints(1025), 16),
        lambda: cache.reserve(host, *state, listed.long(), listed, 16),
        lambda: cache.reserve(host, tables, lengths[:2], refs, listed, listed, 16),
        lambda: cache.reserve(host, *state, listed, listed, 16, missing=ints(2)),
        lambda: cache.fork(host, pool[:, :2], *state, listed, listed, 16),
        lambda: cache.fork(host, pool.transpose(1, 2), *state, listed, listed, 16),
        lambda: cache.fork(host, pool[:1].expand(2, 3, 16), *state, listed, listed, 16),
        lambda: cache.fork(host, pool, *state, listed, ints(3), 16),
        lambda: cache.free(host, *state, ints(2, 2), 16),
        lambda: cache.compact(host, pool, tables, refs, out=(tables,)),
        lambda: cache.compact(host, pool, tables, refs, out=(tables, ints(4))),
        lambda: cache.compact(host, pool, tables.t(), refs),
        lambda: cache.copy_pages(host, pool, ints(2, 3)),
        lambda: cache.copy_pages(host, pool[0], ints(2, 2)),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i}")
    for call in (lambda: cache.reserve(host, *state, listed, listed, 0), lambda: cache.fork(host, pool, *state, listed, listed, 0),
                 lambda: cache.free(host, *state, listed, 1 << 17), lambda: cache.copy_pages(host, pool[:, :, :3].contiguous(), ints(1, 2))):
        with pytest.raises(LsxError):
            call()
    with pytest.raises(LsxError, match="65536"):
        cache.free(host, *state, ints(65537), 16)
    for call in (lambda: cache.reserve(host, *state, listed, listed, 16), lambda: cache.fork(host, pool, *state, listed, listed, 16),
                 lambda: cache.free(host, *state, listed, 16), lambda: cache.compact(host, pool, tables, refs),
                 lambda: cache.copy_pages(host, pool, ints(2, 2))):
        with pytest.raises(LsxError, match="context"):
            call()


def test_pages_of_nothing_and_calls_beyond_the_grid(host):
    _, tables, lengths = held()
    for shape in ((3, 0, 2, 18 * 64), (3, 2, 0, 18 * 64), (3, 2, 2, 0)):
        with pytest.raises(ValueError, match="pages"):
            cache.attention(host, torch.zeros(4, 2, shape[3] // 18), torch.zeros(shape, dtype=torch.uint8), tables, lengths)
    address = 1 << 20
    for rows, heads, word in ((1 << 16, 1 << 15, b"context"), ((1 << 16) + 1, 1 << 15, b"rows of heads"), (1 << 26, 33, b"rows of heads")):
        view = CacheView(pages=address, page_count=3, page_size=32, kv_heads=heads, head_dim=64, tables=address, table_rows=4,
                         table_width=5, lengths=address)
        listed = CacheRows(rows=rows, sequences=4, starts=address)
        assert lib.lsx_cache_append_device(None, C.byref(view), C.byref(listed), address, address, 0, 0, 0, 0, 0, None) != 0
        assert word in lib.lsx_last_error()


def test_calls_of_nothing(host):
    x = torch.zeros(0, 2, 64)
    cache.append(host, x, x, *held(), sequences=ints(0))
    assert cache.attention(host, x, *held(), sequences=ints(0)).shape == x.shape
    cache.free(host, ints(4, 5), ints(4), ints(3), ints(0), 16)
    cache.copy_pages(host, torch.zeros(2, 3, 16), ints(0, 2))


def test_the_library_checks_its_own(host):
    address = 1 << 20
    good = dict(pages=address, page_count=3, page_size=32, kv_heads=2, head_dim=64, tables=address, table_rows=4, table_width=5,
                lengths=address)

    def attend(rows=dict(rows=4, sequences=4), heads=4, scale=1.0, **change):
        view, listed = CacheView(**{**good, **change}), CacheRows(**rows)
        return lib.lsx_cache_attention_device(None, C.byref(view), C.byref(listed), address, 0, heads, 256, 64, scale, address, 256,
                                              64, address, 1 << 30, None)

    assert attend() != 0 and b"context" in lib.lsx_last_error()
    for change in (dict(pages=None), dict(pages=address + 8), dict(page_size=24), dict(page_size=0), dict(head_dim=96),
                   dict(head_dim=320), dict(kv_heads=0), dict(kv_heads=3), dict(page_count=0), dict(page_count=1 << 32),
                   dict(table_width=0), dict(table_width=1 << 30), dict(tables=None), dict(lengths=None), dict(scale=float("nan")),
                   dict(scale=float("inf")), dict(heads=0), dict(rows=dict(rows=0, sequences=4)),
                   dict(rows=dict(rows=5, sequences=5)), dict(rows=dict(rows=5, sequences=4))):
        assert attend(**change) == 1 and b"context" not in lib.lsx_last_error(), change
    pool = dict(data=address, layers=2, layer_bytes=480, page_bytes=48, page_count=10)
    for change in (dict(data=None), dict(layers=0), dict(layer_bytes=472), dict(layer_bytes=464), dict(page_bytes=40),
                   dict(page_count=0), dict(data=address + 8)):
        assert lib.lsx_cache_copy_device(None, C.byref(CachePool(**{**pool, **change})), address, 1, None) == 1
        assert b"context" not in lib.lsx_last_error(), change
    assert lib.lsx_cache_copy_device(None, C.byref(CachePool(**pool)), address, 1, None) == 1
    assert b"context" in lib.lsx_last_error()
