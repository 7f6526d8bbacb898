"""Packed attention, the 4-bit cache and page copies without a GPU: refusals that come before any launch, the page
allocator's sharing, forking and compacting, and the 64-bit reference against differences."""
import ctypes
import math

import pytest
import torch

import b200_llama as B
import packed_reference as R

P = ctypes.c_void_p(16)   # a non-null, aligned address that no refused call touches


def test_packed_attention_refusals():
    f = B.lib().b200_attention_packed
    call = lambda q=P, k=P, v=P, o=P, cu=P, n=1, rows=8, h=4, hk=2, hs=64, ldq=256, ldk=128, ldv=128, ldo=256, dt=1, impl=0: f(
        q, k, v, o, None, cu, n, rows, h, hk, hs, ldq, ldk, ldv, ldo, dt, impl, None)
    assert call(q=None) == 1 and call(cu=None) == 1 and call(impl=5) == 1
    assert call(h=3) == 2 and call(hk=0) == 2 and call(hs=40) == 2 and call(rows=-1) == 2 and call(ldk=100) == 2
    assert call(dt=7) == 3
    assert call(rows=0, q=None) == 0 and call(n=0, q=None) == 0       # nothing to do
    g = B.lib().b200_attention_packed_backward
    assert g(P, P, P, P, P, P, P, P, P, None, P, 1, 8, 4, 2, 64, 256, 128, 128, 256, 256, 256, 128, 128, 1, 0, None) == 1
    assert g(P, P, P, P, P, P, P, P, P, P, P, 1, 8, 4, 2, 64, 256, 128, 128, 256, 256, 256, 64, 128, 1, 0, None) == 2


def test_kv4_refusals():
    lib = B.lib()
    app = lambda k=P, codes=P, table=P, n=1, rows=4, hk=2, hs=64, ldk=128, pages=4, page=16, width=2, dt=1: lib.b200_kv4_append(
        k, P, codes, P, table, P, None, n, rows, hk, hs, ldk, 128, pages, page, width, dt, None)
    assert app(k=None) == 1 and app(table=None) == 1 and app(hs=20) == 2 and app(page=0) == 2 and app(ldk=64) == 2
    assert app(dt=5) == 3 and app(codes=ctypes.c_void_p(18)) == 4 and app(rows=0, k=None) == 0
    dec = lambda q=P, scratch=P, nbytes=1 << 30, b=1, h=4, hk=2, hs=64, ldq=256, impl=0: lib.b200_attention_decode_kv4(
        q, P, P, P, P, P, scratch, nbytes, b, h, hk, hs, ldq, 256, 4, 16, 2, 1, impl, None)
    assert dec(q=None) == 1 and dec(h=3) == 2 and dec(ldq=8) == 2 and dec(b=-1) == 2 and dec(impl=9) == 1
    assert dec(b=0, q=None) == 0 and dec(scratch=ctypes.c_void_p(8)) == 4
    n = ctypes.c_size_t(0)
    assert lib.b200_attention_decode_kv4_scratch_bytes(4, 4, 3, 64, ctypes.byref(n)) == 2
    assert lib.b200_attention_decode_kv4_scratch_bytes(4, 4, 2, 64, None) == 1


def test_kv4_refusals_by_size():
    lib = B.lib()
    n = ctypes.c_size_t(0)
    size = lambda batch=4, h=4, hk=2, hs=64, page=16, width=2, dt=1, out=ctypes.byref(n): (
        lib.b200_attention_decode_kv4_scratch_bytes_for(batch, h, hk, hs, page, width, dt, out))
    assert size(h=3) == 2 and size(batch=-1) == 2 and size(page=0) == 2 and size(width=-1) == 2 and size(out=None) == 1
    dec = lambda page=16, width=2, b=1: lib.b200_attention_decode_kv4(
        P, P, P, P, P, P, P, 1 << 30, b, 4, 2, 64, 256, 256, 4, page, width, 1, 0, None)
    assert dec(page=1 << 30) == 2                       # more rows than a page may have
    assert dec(page=1 << 20, width=1 << 14, b=1 << 12) == 2   # page tables that are too long together


def test_copy_pages_refusals():
    f = B.lib().b200_copy_pages
    call = lambda pool=P, planes=2, pages=4, heads=2, page=16, row=128, src=P, n=1, table=None, entries=0, pmap=None: f(
        pool, planes, pages, heads, page, row, src, P, None, n, table, entries, pmap, None)
    assert call(pool=None) == 1 and call(src=None) == 1 and call(table=P, entries=4) == 1
    assert call(planes=0) == 2 and call(n=-1) == 2 and call(row=0) == 2 and call(page=1 << 30) == 2
    assert call(n=0, pool=None) == 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 128).bfloat16()
    cu = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: B.attention_packed(x, x, x, cu, 2), lambda: B.copy_pages(torch.zeros(2, 4, 2, 16, 64), [0], [1])):
        with pytest.raises(B.B200Error) as e:
            call()
        assert e.value.status == 1


def test_allocator_shares_and_forks():
    a = B.PageAllocator(8)
    x = a.alloc(3)
    child, copies = a.fork(x, 40, 16)               # two full pages, 8 rows of the third
    assert child[:2] == x[:2] and child[2] not in x and copies == [(x[2], child[2], 8)]
    assert [a.refs(p) for p in x] == [2, 2, 1] and a.free_pages == 4
    whole, none = a.fork(x, 32, 16)                 # ends with a page: nothing to copy
    assert whole == x[:2] and none == [] and a.refs(x[0]) == 3
    assert a.fork(x, 0, 16) == ([], [])
    a.free(x)
    assert a.free_pages == 5 and a.refs(x[2]) == 0 and a.refs(x[0]) == 2
    a.free(child)
    a.free(whole)
    assert a.free_pages == 8
    with pytest.raises(B.B200Error):
        a.free([x[0]])                              # not held any more
    y = a.alloc(2)
    with pytest.raises(B.B200Error):
        a.free([y[0], y[0]])                        # once per holder: nothing is given back
    assert a.refs(y[0]) == 1
    with pytest.raises(B.B200Error):
        a.fork(y, 33, 16)
    full = a.alloc(6)
    with pytest.raises(B.B200Error) as e:
        a.fork(y, 5, 16)                            # no page for the partly filled one: nothing is shared
    assert e.value.status == 5 and a.refs(y[0]) == 1
    with pytest.raises(B.B200Error):
        a.share([full[0], 99])
    assert a.refs(full[0]) == 1


def test_allocator_compacts():
    a = B.PageAllocator(10)
    x, y, z = a.alloc(3), a.alloc(3), a.alloc(2)
    a.share([z[1]])
    a.free(x)
    src, dst, page_map = a.compact()
    live = sorted(page_map[p] for p in y + z)
    assert live == [0, 1, 2, 3, 4] and len(set(dst)) == len(dst) and not set(src) & set(dst)
    assert all(page_map[s] == d for s, d in zip(src, dst)) and a.refs(page_map[z[1]]) == 2
    assert a.free_pages == 5 and a.alloc(1) == [5]
    assert a.compact()[0] == []                     # already compact
    a.free([page_map[p] for p in y + z])
    assert a.refs(page_map[z[1]]) == 1


def test_allocator_takes_page_numbers_of_any_integer_kind():
    a = B.PageAllocator(6)
    x = torch.tensor(a.alloc(4), dtype=torch.int32)
    assert a.refs(x[1]) == 1
    a.free(x[2:])                                   # a row of a page table, its elements 0-d tensors
    assert a.free_pages == 4
    a.share(x[:1])
    child, copies = a.fork(x[:2], 20, 16)
    assert child[0] == int(x[0]) and a.refs(int(x[0])) == 3 and copies[0][0] == int(x[1])
    assert all(type(p) is int for p in child)
    a.free(x[:2].numpy())
    a.free([x[0]])
    a.free(child)
    assert a.free_pages == 6 and sorted(a.alloc(6)) == list(range(6))
    with pytest.raises(B.B200Error):
        a.free(torch.tensor([6]))


@pytest.fixture
def launches(monkeypatch):
    """The arguments of every call that would go to the library, with tensors of the host in the place of the device's."""
    made = []
    monkeypatch.setattr(B, "_device_of", lambda what, names, *tensors: torch.device("cpu"))
    monkeypatch.setattr(B, "_page_list", lambda what, name, x, dev: torch.as_tensor(x, dtype=torch.int32))
    monkeypatch.setattr(B, "_call", lambda dev, fn, *args: made.append(args))
    return made


def test_compact_rewrites_the_table_whatever_the_pools_hold(launches):
    full, empty = torch.zeros(2, 6, 2, 4, 8), torch.zeros(0, 6, 2, 4, 8)
    table = torch.tensor([[5, 4]], dtype=torch.int32)
    for pools, copies in (([full, empty], [2]), ([empty, full], [2]), ([full, full], [2, 2]), ([empty], [0])):
        launches.clear()
        B.compact_pages(pools, [5, 4], [0, 1], table, [0, 1, 2, 3, 1, 0])
        assert [a[9] for a in launches] == copies             # copies of each launch
        assert [a[11] for a in launches] == [0] * (len(copies) - 1) + [2]   # and table entries: once, with the last
        assert all(min(a[1:6]) > 0 for a in launches)


def test_a_refused_compaction_moves_nothing(launches):
    good, other = torch.zeros(2, 6, 2, 4, 8), torch.zeros(2, 6, 2, 4, 16)[..., ::2]
    table = torch.tensor([[5, 4]], dtype=torch.int32)
    with pytest.raises(B.B200Error):
        B.compact_pages([good, other], [5], [0], table, [0, 1, 2, 3, 4, 0])      # the second pool is not contiguous
    with pytest.raises(B.B200Error):
        B.compact_pages([good, good], [5], [0], table, [0, 1, 2, 3, 4])          # the map names five pages of six
    assert not launches


def test_decode_scratch_goes_by_the_device_of_the_tensors(monkeypatch):
    """Devices may differ in their number of SMs, and the current one need not be the tensors'."""
    current = [0]

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *exc):
            current[0] = self.before

    class Lib:
        @staticmethod
        def b200_attention_decode_kv4_scratch_bytes_for(*args):
            args[-1]._obj.value = 1000 * (current[0] + 1)
            return 0

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(B, "lib", lambda: Lib)
    sizes = (2, 4, 2, 64, 16, 40, 1)
    B._kv4_scratch_bytes.cache_clear()
    try:
        assert [B._kv4_scratch_bytes(d, *sizes) for d in (0, 1, 0, 1)] == [1000, 2000, 1000, 2000]
    finally:
        B._kv4_scratch_bytes.cache_clear()
    assert current == [0]


def test_pitches_and_pages_past_32_bits_are_refused(launches):
    """Sizes go to the library in 32 bits; what does not fit is refused, not cut to its low half."""
    wide = torch.empty(2, (1 << 32) + 64, dtype=torch.bfloat16, device="meta")[:, :64]
    with pytest.raises(B.B200Error) as e:
        B._rows("x", "q", wide, 64)
    assert e.value.status == 2
    assert B._rows("x", "q", torch.empty(2, (1 << 31) - 1, dtype=torch.uint8, device="meta")[:, :64], 64) == (1 << 31) - 1
    pool = torch.empty(1, 2, 1, 1, (1 << 32) + 64, dtype=torch.uint8, device="meta")
    with pytest.raises(B.B200Error) as e:
        B.copy_pages(pool, [0], [1])
    assert e.value.status == 2 and not launches


def test_reference_gradient_against_differences():
    g = torch.Generator().manual_seed(0)
    lens, heads, kv, hs = [5, 1, 7], 4, 2, 8
    q, k, v, d_o = (torch.randn(13, n * hs, generator=g, dtype=torch.float64) for n in (heads, kv, kv, heads))
    R.U[torch.float64] = 0.0
    try:
        grads, _ = R.backward(q, k, v, d_o, lens, heads, kv)
        value = lambda a, b, c: float((R.forward(a, b, c, lens, heads, kv)[0] * d_o).sum())
        h = 1e-6
        for i, grad in enumerate(grads):
            d = torch.randn(grad.shape, generator=g, dtype=torch.float64)
            up, down = [q, k, v], [q, k, v]
            up[i], down[i] = up[i] + h * d, down[i] - h * d
            diff = (value(*up) - value(*down)) / (2 * h)
            assert math.isclose(diff, float((grad * d).sum()), rel_tol=1e-7, abs_tol=1e-7)
    finally:
        del R.U[torch.float64]
