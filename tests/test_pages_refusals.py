"""What the paged operators and the chain verification refuse, before any CUDA call (no GPU is touched)."""
import ctypes as C

import pytest
import torch

from seedplane_b200 import _native as N
from seedplane_b200.build import build

PTR = 4096                                               # never dereferenced: every call here is refused


@pytest.fixture(scope="module")
def lib():
    build()
    return N.load()


def pages(**change):
    p = dict(k_dev=PTR, v_dev=PTR, page_stride=2 * 16 * 64, head_stride=16 * 64, slot_stride=64, n_pages=9, page_size=16,
             kv_heads=2, head_dim=64, dtype=N.SP_F16, status_dev=PTR)
    return N.SpPages(**(p | change))


def batch(**change):
    b = dict(batch=3, tokens=3, max_q=1, q_start_dev=None, lens_dev=PTR, tables_dev=PTR, table_stride=4, table_width=4,
             prefix_dev=PTR, prefix_len=20)
    return N.SpPageBatch(**(b | change))


def append(lib, p, b, heads=4, qkv=PTR, dtype=N.SP_F16, xs=8 * 64, rope=PTR, positions=100, rot=64, q=PTR, qs=4 * 64):
    return lib.sp_pages_append(0, p, b, heads, qkv, dtype, xs, None, rope, positions, rot, 0, None, q, qs, None)


def attention(lib, p, b, heads=4, q=PTR, dtype=N.SP_F16, qs=4 * 64, scale=0.125, out=PTR, os_=4 * 64, ws=PTR, size=1 << 40):
    return lib.sp_pages_attention(0, p, b, heads, q, dtype, qs, scale, out, os_, None, ws, size, None)


BAD_PAGES = [(dict(head_dim=96), N.SP_ERR_UNSUPPORTED), (dict(head_dim=32), N.SP_ERR_UNSUPPORTED),
             (dict(dtype=N.SP_F32), N.SP_ERR_UNSUPPORTED), (dict(dtype=7), N.SP_ERR_UNSUPPORTED),
             (dict(page_size=0), N.SP_ERR_INVALID), (dict(n_pages=-1), N.SP_ERR_INVALID), (dict(n_pages=0), N.SP_ERR_INVALID),
             (dict(kv_heads=0), N.SP_ERR_INVALID), (dict(kv_heads=3), N.SP_ERR_INVALID), (dict(k_dev=None), N.SP_ERR_INVALID),
             (dict(v_dev=PTR + 2), N.SP_ERR_INVALID), (dict(slot_stride=65), N.SP_ERR_INVALID),
             (dict(page_size=1 << 30), N.SP_ERR_CAPACITY)]
BAD_BATCH = [(dict(batch=0), N.SP_ERR_INVALID), (dict(batch=-1), N.SP_ERR_INVALID), (dict(max_q=0), N.SP_ERR_INVALID),
             (dict(tokens=-1), N.SP_ERR_INVALID), (dict(lens_dev=None), N.SP_ERR_INVALID), (dict(tables_dev=None), N.SP_ERR_INVALID),
             (dict(table_stride=3), N.SP_ERR_INVALID), (dict(prefix_dev=None), N.SP_ERR_INVALID),
             (dict(prefix_len=-1), N.SP_ERR_INVALID), (dict(prefix_len=2 ** 31 - 1), N.SP_ERR_CAPACITY),
             (dict(tokens=2 ** 30), N.SP_ERR_CAPACITY), (dict(batch=2 ** 30), N.SP_ERR_CAPACITY),
             (dict(batch=2 ** 20, tokens=2 ** 20, max_q=2 ** 20), N.SP_ERR_CAPACITY)]


@pytest.mark.parametrize("change,code", BAD_PAGES)
def test_bad_pages(lib, change, code):
    assert append(lib, pages(**change), batch()) == code
    assert attention(lib, pages(**change), batch()) == code
    assert lib.sp_pages_attention_workspace(pages(**change), batch(), 4, N.SP_F16) == code
    assert lib.sp_last_error()


@pytest.mark.parametrize("change,code", BAD_BATCH)
def test_bad_batches(lib, change, code):
    assert append(lib, pages(), batch(**change)) == code
    assert attention(lib, pages(), batch(**change)) == code


def test_bad_arguments(lib):
    p, b = pages(), batch()
    assert append(lib, None, b) == append(lib, p, None) == N.SP_ERR_INVALID
    for bad in (dict(qkv=None), dict(rope=None), dict(q=None), dict(xs=8 * 64 - 1), dict(qs=4 * 64 - 1), dict(rot=0), dict(rot=63),
                dict(rot=66), dict(positions=0), dict(heads=0), dict(heads=3)):
        assert append(lib, p, b, **bad) == N.SP_ERR_INVALID, bad
    assert append(lib, p, b, dtype=N.SP_BF16) == N.SP_ERR_UNSUPPORTED
    for bad in (dict(q=None), dict(out=None), dict(qs=100), dict(os_=4 * 64 + 1), dict(q=PTR + 8), dict(scale=0.0),
                dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf"))):
        assert attention(lib, p, b, **bad) == N.SP_ERR_INVALID, bad
    longer = batch(prefix_len=20000)                     # key ranges whose results are joined need a workspace
    assert lib.sp_pages_attention_workspace(p, longer, 4, N.SP_F16) > 8
    for bad in (dict(size=8), dict(ws=None), dict(ws=PTR + 4)):
        assert attention(lib, p, longer, **bad) == N.SP_ERR_INVALID, bad
    assert attention(lib, p, b, dtype=N.SP_BF16) == N.SP_ERR_UNSUPPORTED
    assert attention(lib, pages(dtype=N.SP_BF16), b, dtype=N.SP_F32) == N.SP_ERR_UNSUPPORTED
    # nothing to do is fine, whatever the pointers
    assert append(lib, p, batch(tokens=0), qkv=None) == N.SP_OK
    assert attention(lib, p, batch(tokens=0, batch=0, lens_dev=None), q=None) == N.SP_OK


def chains(lib, B=2, n=3, V=100, target=PTR, ld=100, draft=PTR, dld=100, dtype=0, tokens=PTR, u=PTR, out=PTR, acc=PTR, ws=PTR,
           size=1 << 40):
    return lib.sp_accept_chains(0, B, n, V, target, (n + 1) * ld, ld, draft, n * dld, dld, dtype, tokens, None, u, None, out, acc,
                                ws, size, None)


def test_bad_chains(lib):
    for bad in (dict(B=-1), dict(V=0), dict(target=None), dict(tokens=None), dict(u=None), dict(out=None), dict(acc=None),
                dict(ld=99), dict(dld=99), dict(ws=None), dict(ws=PTR + 8), dict(size=10)):
        assert chains(lib, **bad) == N.SP_ERR_INVALID, bad
    assert chains(lib, n=65) == chains(lib, n=-1) == chains(lib, B=10 ** 6, n=64, V=2 * 10 ** 6) == N.SP_ERR_CAPACITY
    assert chains(lib, dtype=3) == N.SP_ERR_UNSUPPORTED
    assert chains(lib, B=0, target=None) == N.SP_OK
    assert lib.sp_accept_chains_workspace(1, 65, 10) == N.SP_ERR_CAPACITY
    assert lib.sp_accept_chains_workspace(4, 3, 151936) > 0


def test_passes_without_an_engine(lib):
    one = (N.SpPages * 1)(pages())
    assert lib.sp_forward_pages(None, one, batch(), PTR, None, PTR, None) == N.SP_ERR_INVALID
    assert lib.sp_forward_pages(None, None, None, None, None, None, None) == N.SP_ERR_INVALID
    assert lib.sp_decode_pages(None, one, batch(), PTR, 1, PTR, None) == N.SP_ERR_INVALID
    assert lib.sp_decode_pages(None, one, batch(), PTR, 0, PTR, None) == N.SP_ERR_INVALID
    assert lib.sp_decode_pages(None, one, batch(max_q=2, tokens=6), PTR, 1, PTR, None) == N.SP_ERR_INVALID
    assert lib.sp_decode_pages(None, one, batch(q_start_dev=PTR), PTR, 1, PTR, None) == N.SP_ERR_INVALID


def test_python_checks_come_before_the_library():
    from seedplane_b200 import paged, speculative
    k = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        paged.PagedKV.wrap(k, k)                         # not on a CUDA device
    with pytest.raises(ValueError):
        paged.PagedKV.wrap(k, k[:3])
    with pytest.raises(ValueError):
        paged.PagedKV.wrap(k.float(), k.float())
    lens, tables = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32)
    with pytest.raises(ValueError):
        paged.PageBatch(tables[:2], lens)
    with pytest.raises(ValueError):
        paged.PageBatch(tables.long(), lens)
    with pytest.raises(ValueError):
        paged.PageBatch(tables, lens, q_start=torch.zeros(4, dtype=torch.int32))      # no `tokens`
    with pytest.raises(ValueError):
        paged.PageBatch(tables, lens, q_start=torch.zeros(3, dtype=torch.int32), tokens=3)
    with pytest.raises(ValueError):
        paged.PageBatch(tables.t().contiguous().t(), lens)
    x = torch.zeros(2, 3, 10)
    with pytest.raises(ValueError):
        speculative.accept_chains(x, None, torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.float64))
