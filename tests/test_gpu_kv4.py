"""The 4-bit key/value cache: quantisation to the bit, read back, decode attention, page copies, and a run of them."""
import ctypes
import math

import pytest
import torch

import b200_llama as B

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
U32 = 2.0 ** -24


def cu_of(lens):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=DEV)


def tables(lens, page, seed=0, spare=2):
    need = [max(1, -(-n // page)) for n in lens]
    total = sum(need) + spare
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    width, rows, at = max(need), [], 0
    for n in need:
        rows.append(perm[at:at + n] + [-1] * (width - n))   # unused entries name no page
        at += n
    return torch.tensor(rows, dtype=torch.int32, device=DEV), total


def quantise(x):
    """The definition, one rounding after the other, in fp32 with true divisions."""
    x = x.float()
    lo = x.amin(-1, keepdim=True)
    b = lo.view(torch.int32)
    cut = b & -65536
    lo = torch.where((b < 0) & (cut != b), cut + 65536, cut).view(torch.float32)
    sc = (x.amax(-1, keepdim=True) - lo) / torch.full_like(lo, 15.0)
    b = sc.view(torch.int32)
    cut = b & -65536
    sc = torch.where(cut != b, cut + 65536, cut).view(torch.float32)
    codes = torch.where(sc > 0, torch.round((x - lo) / torch.where(sc > 0, sc, torch.ones_like(sc))), torch.zeros_like(x))
    return codes.clamp(0, 15), sc, lo


@pytest.mark.parametrize("hs,hk,page,dtype,lens,before", [
    (128, 8, 64, torch.bfloat16, [1, 200, 63, 0, 64], [0, 5, 1, 7, 64]),
    (64, 2, 16, torch.bfloat16, [33], [0]),
    (48, 6, 12, torch.float32, [1, 1, 1, 1], [11, 12, 0, 100]),
    (32, 1, 64, torch.float32, [300], [77]),
    (16, 3, 7, torch.bfloat16, [20, 21], [0, 0]),
])
def test_append_and_read(hs, hk, page, dtype, lens, before):
    g = torch.Generator(device=DEV).manual_seed(1)
    T = sum(lens)
    kv = torch.randn(T, 2 * hk * hs, generator=g, device=DEV).to(dtype)
    kv[0, :hs] = 0.25                       # a row of equal elements: scale 0
    kv[T - 1, :hs] = torch.linspace(-3, 3, hs, device=DEV).to(dtype)
    if T > 20:                              # exact ties: (k + 1/2) steps of 1/4, and of the smallest and largest scales
        kv[1, :hs] = (torch.arange(hs, device=DEV) % 31).to(dtype) / 8
        kv[2, :hs] = kv[1, :hs] * 2.0 ** -124
        kv[3, :hs] = kv[1, :hs] * 2.0 ** 124
        kv[4, :hs] = -kv[1, :hs]
    k, v = kv[:, :hk * hs], kv[:, hk * hs:]
    table, n_pages = tables([n + b for n, b in zip(lens, before)], page)
    codes, params = B.new_kv4_pages(1, n_pages, hk, page, hs)
    codes.fill_(0xAB)
    params.fill_(5.0)
    bt = torch.tensor(before, dtype=torch.int32, device=DEV)
    B.kv4_append(k, v, codes[0], params[0], table, cu_of(lens), bt)
    assert B.device_status() == 0
    want_c, want_p = torch.full_like(codes[0], 0xAB), torch.full_like(params[0], 5.0)
    t = 0
    back = []
    for s, n in enumerate(lens):
        for i in range(n):
            pos = before[s] + i
            pg, r = int(table[s, pos // page]), pos % page
            for half, x in enumerate((k, v)):
                c, sc, lo = quantise(x[t].view(hk, hs))
                cu8 = c.to(torch.uint8)
                want_c[half, pg, :, r] = cu8[:, 0::2] | (cu8[:, 1::2] << 4)
                want_p[half, pg, :, r] = torch.cat((sc, lo), -1).bfloat16()
                # half a step; the quotient, below 16, is rounded twice (x - lo, the division): 32 U32 steps; this line's
                # own product, sum and difference round numbers below |lo| + 16 sc: 3 U32 each time
                slack = U32 * (32 * sc + 3 * (lo.abs() + 16 * sc))
                assert bool(((c * sc + lo - x[t].view(hk, hs).float()).abs() <= 0.5 * sc + slack).all())
                back.append((c * sc + lo).to(dtype).view(-1))
            t += 1
    assert torch.equal(codes[0], want_c)
    assert torch.equal(params[0], want_p)   # rows that were not appended stay as they were
    rk, rv = B.kv4_read(codes[0], params[0], table, cu_of(lens), bt, T, dtype=dtype)
    assert torch.equal(rk, torch.stack(back[0::2])) and torch.equal(rv, torch.stack(back[1::2]))


def test_append_rows_that_are_not_finite():
    hs, hk = 64, 2
    k = torch.randn(6, hk * hs, device=DEV).bfloat16()
    v = k.clone()
    k[0, 3], k[1, 70], k[2, 0], v[3, 127] = math.nan, math.inf, -math.inf, math.nan
    k[4, :2] = torch.tensor([3.3e38, -3.3e38], device=DEV).bfloat16()   # the spread overflows
    table, n_pages = tables([6], 16)
    codes, params = B.new_kv4_pages(1, n_pages, hk, 16, hs)
    B.kv4_append(k, v, codes[0], params[0], table, cu_of([6]))
    rk, rv = B.kv4_read(codes[0], params[0], table, cu_of([6]), None, 6)
    bad_k = torch.zeros(6, hk, dtype=torch.bool, device=DEV)
    bad_k[0, 0] = bad_k[1, 1] = bad_k[2, 0] = bad_k[4, 0] = True
    bad_v = torch.zeros_like(bad_k)
    bad_v[3, 1] = True
    assert torch.equal(rk.view(6, hk, hs).isnan().all(-1), bad_k) and torch.equal(rk.view(6, hk, hs).isnan().any(-1), bad_k)
    assert torch.equal(rv.view(6, hk, hs).isnan().all(-1), bad_v) and torch.equal(rv.view(6, hk, hs).isnan().any(-1), bad_v)


def test_append_without_a_place_is_skipped_and_reported():
    hs, hk, page = 64, 1, 16
    k = torch.randn(40, hs, device=DEV).bfloat16()
    table = torch.tensor([[0, 99], [1, -1]], dtype=torch.int32, device=DEV)   # pool of 3 pages
    codes, params = B.new_kv4_pages(1, 3, hk, page, hs)
    params.fill_(9.0)
    B.kv4_append(k, k, codes[0], params[0], table, cu_of([20, 20]))
    with pytest.raises(B.B200Error) as e:
        B.device_status()
    assert e.value.status == 1
    assert B.device_status() == 0
    assert bool((params[0, :, 2] == 9).all()) and not bool((params[0, :, :2] == 9).any())
    # past the page table
    B.kv4_append(k[:1], k[:1], codes[0], params[0], table[:1], cu_of([1]), torch.tensor([32], dtype=torch.int32, device=DEV))
    with pytest.raises(B.B200Error):
        B.device_status()


def cache(lens, hk, page, hs, seed=0):
    """A cache filled at random; rows behind every sequence's end hold NaN parameters."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    table, n_pages = tables(lens, page, seed)
    codes = torch.randint(0, 256, (2, n_pages, hk, page, hs // 2), generator=g, device=DEV, dtype=torch.uint8)
    params = torch.full((2, n_pages, hk, page, 2), math.nan, device=DEV).bfloat16()
    for s, n in enumerate(lens):
        for i in range(-(-n // page)):
            r = min(page, n - i * page)
            sc = torch.rand(2, hk, r, generator=g, device=DEV) * 0.3 + 0.05
            lo = -7.5 * sc + 0.3 * torch.randn(2, hk, r, generator=g, device=DEV)
            params[:, int(table[s, i]), :, :r] = torch.stack((sc, lo), -1).bfloat16()
    return codes, params, table


def decode_reference(q, codes, params, table, lens, heads):
    """fp64 output and the bound of a kernel.  Scores and sums are fp32; in the bf16 form query elements stand to half a
    step of 1/32512 of the head's largest and the weights scale * p of the codes to half a step of 1/65535 of a reference
    that is at most 8 times the largest weight (4 for p, 2 for the scale).
      |do| <= U|o| + (2 ds + (n + 16) U32) sum p (|lo| + 15 scale) + n 2^-14 max(p) max(scale) 15,
      ds <= (hs + 16) U32 sum|q| (|lo| + 15 scale) / sqrt(hs) + 2^-16 max|q| hs 15 scale / sqrt(hs)"""
    hk, page, hs = codes.shape[2], codes.shape[3], codes.shape[4] * 2
    group = heads // hk
    out = torch.zeros(len(lens), heads, hs, dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(out)
    small = q.dtype == torch.bfloat16
    for b, n in enumerate(lens):
        if n == 0:
            continue
        at = torch.arange(n, device=DEV)
        pg, r = table[b].long()[at // page], at % page
        for j in range(hk):
            rows, mags = [], []
            for half in range(2):
                c = codes[half, pg, j, r]
                prm = params[half, pg, j, r].double()
                x = torch.stack((c & 15, c >> 4), -1).view(n, hs).double()
                rows.append(x * prm[:, :1] + prm[:, 1:])
                mags.append(15 * prm[:, :1] + prm[:, 1:].abs())
            ksc, vsc = params[0, pg, j, r, :1].double(), params[1, pg, j, r, :1].double()
            hd = slice(j * group, (j + 1) * group)
            Q = q[b].view(heads, hs)[hd].double()
            s = Q @ rows[0].T / math.sqrt(hs)
            p = torch.softmax(s, -1)
            ds = (hs + 16) * U32 * Q.abs().sum(-1, keepdim=True) * mags[0].T / math.sqrt(hs)
            if small:
                ds = ds + 2.0 ** -16 * Q.abs().amax(-1, keepdim=True) * hs * 15 * ksc.T / math.sqrt(hs)
            ds = ds.max(-1, keepdim=True).values
            out[b, hd] = p @ rows[1]
            bound[b, hd] = U[q.dtype] * out[b, hd].abs() + ((2 * ds + (n + 16) * U32) * p) @ mags[1].expand(n, hs)
            if small:
                bound[b, hd] += n * 2.0 ** -14 * p.amax(-1, keepdim=True) * vsc.max() * 15
    return out.view(len(lens), -1), bound.view(len(lens), -1) + 1e-30


DECODE = [  # lens, heads, kv_heads, hs, page, dtype
    ([1], 6, 6, 48, 16, torch.float32),
    ([5, 0, 700], 4, 2, 64, 12, torch.float32),
    ([300, 1], 3, 1, 16, 7, torch.bfloat16),
    ([1], 4, 1, 128, 64, torch.bfloat16),
    ([500], 32, 8, 128, 64, torch.bfloat16),
    ([127, 128, 129, 0, 1, 16, 17], 4, 4, 64, 16, torch.bfloat16),
    ([3000, 2, 1111], 12, 2, 128, 128, torch.bfloat16),
    ([400, 77], 8, 1, 64, 32, torch.bfloat16),
    ([350, 64], 20, 1, 128, 64, torch.bfloat16),
    ([90] * 70, 2, 1, 64, 16, torch.bfloat16),
    ([200, 33], 5, 1, 128, 20, torch.bfloat16),
    ([9000], 2, 2, 128, 64, torch.bfloat16),
    ([300, 47], 4, 2, 128, 48, torch.bfloat16),
    ([513, 96], 8, 8, 64, 96, torch.bfloat16),
    ([1000, 256, 257], 7, 1, 128, 256, torch.bfloat16),
]


@pytest.mark.parametrize("impl", [0, 2])
@pytest.mark.parametrize("lens,heads,hk,hs,page,dtype", DECODE)
def test_decode(lens, heads, hk, hs, page, dtype, impl):
    codes, params, table = cache(lens, hk, page, hs, seed=len(lens))
    q = torch.randn(len(lens), heads * hs, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).to(dtype)
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    o = B.attention_decode_kv4(q, codes, params, table, ctx, heads, impl=impl)
    assert B.device_status() == 0
    want, bound = decode_reference(q, codes, params, table, lens, heads)
    err = (o.double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    for _ in range(2):
        assert torch.equal(o, B.attention_decode_kv4(q, codes, params, table, ctx, heads, impl=impl))


@pytest.mark.parametrize("heads,hk,hs,dtype", [(8, 2, 128, torch.bfloat16), (20, 1, 64, torch.bfloat16), (6, 3, 48, torch.float32)])
def test_decode_short_and_long_tables(heads, hk, hs, dtype):
    # short tables need no scratch and one kernel; the same rows under longer tables are shared out and joined
    lens = [200, 0, 256, 129, 1]
    codes, params, table = cache(lens, hk, 64, hs, seed=8)
    q = torch.randn(len(lens), heads * hs, generator=torch.Generator(device=DEV).manual_seed(5), device=DEV).to(dtype)
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    n = ctypes.c_size_t(7)
    sizes = (len(lens), heads, hk, hs, 64)
    fn = B.lib().b200_attention_decode_kv4_scratch_bytes_for
    assert fn(*sizes, table.shape[1], B._dt(dtype), ctypes.byref(n)) == 0 and n.value == 0
    long_table = torch.zeros(len(lens), 20, dtype=torch.int32, device=DEV)
    long_table[:, :table.shape[1]] = table
    assert fn(*sizes, 20, B._dt(dtype), ctypes.byref(n)) == 0 and n.value > 0
    want, bound = decode_reference(q, codes, params, table, lens, heads)
    for t in (table, long_table):
        o = B.attention_decode_kv4(q, codes, params, t, ctx, heads, out=torch.full_like(q, float("nan")))
        assert B.device_status() == 0
        assert bool(((o.double() - want).abs() <= bound).all())
    scratch = torch.empty(n.value, dtype=torch.uint8, device=DEV)
    assert torch.equal(o, B.attention_decode_kv4(q, codes, params, long_table, ctx, heads, scratch=scratch))
    with pytest.raises(B.B200Error) as e:
        B.attention_decode_kv4(q, codes, params, long_table, ctx, heads, scratch=scratch[:-16])
    assert e.value.status == 5


@pytest.mark.parametrize("impl", [0, 2])
def test_decode_wide_scores(impl):
    lens, heads, hk, hs, page = [1500, 40], 8, 2, 128, 64
    codes, params, table = cache(lens, hk, page, hs, seed=5)
    q = (torch.randn(2, heads * hs, device=DEV) * 20).bfloat16()
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    o = B.attention_decode_kv4(q, codes, params, table, ctx, heads, impl=impl)
    want, bound = decode_reference(q, codes, params, table, lens, heads)
    assert bool(((o.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("impl", [0, 2])
def test_decode_skips_pages_outside_the_pool(impl):
    lens, heads, hk, hs, page = [200], 4, 1, 128, 64
    codes, params, table = cache(lens, hk, page, hs, seed=7)
    q = torch.randn(1, heads * hs, device=DEV).bfloat16()
    table[0, 1] = 1 << 30
    o = B.attention_decode_kv4(q, codes, params, table, torch.tensor(lens, dtype=torch.int32, device=DEV), heads, impl=impl)
    with pytest.raises(B.B200Error) as e:
        B.device_status()
    assert e.value.status == 1 and bool(torch.isfinite(o.float()).all())
    # lengths that exceed the page table are cut to it, negative ones count as zero
    codes, params, table = cache([128], hk, page, hs, seed=8)
    for n, same in ((1 << 30, 128), (-5, 0)):
        a = B.attention_decode_kv4(q, codes, params, table, torch.tensor([n], dtype=torch.int32, device=DEV), heads, impl=impl)
        b = B.attention_decode_kv4(q, codes, params, table, torch.tensor([same], dtype=torch.int32, device=DEV), heads, impl=impl)
        assert torch.equal(a, b)
    assert B.device_status() == 0


def test_layers_of_odd_size():
    """Pools whose layers are not a multiple of 16 bytes: the second layer begins anywhere on 4 bytes."""
    hk, hs, page = 1, 16, 7
    codes, params = B.new_kv4_pages(2, 3, hk, page, hs)
    assert params[1].data_ptr() % 16
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn(9, hs, generator=g, device=DEV) for _ in range(2))
    table = torch.tensor([[2, 0]], dtype=torch.int32, device=DEV)
    B.kv4_append(k, v, codes[1], params[1], table, cu_of([9]))
    q = torch.randn(1, 2 * hs, generator=g, device=DEV)
    o = B.attention_decode_kv4(q, codes[1], params[1], table, torch.tensor([9], dtype=torch.int32, device=DEV), 2)
    want, bound = decode_reference(q, codes[1], params[1], table, [9], 2)
    assert bool(((o.double() - want).abs() <= bound).all())
    assert bool((codes[0] == 0).all()) and B.device_status() == 0
    with pytest.raises(B.B200Error):
        B.kv4_read(codes[1], params[1], table, cu_of([9]), None, -1)


def test_decode_many_sequences():
    """More sequences than one launch takes."""
    lens = [(i * 7) % 40 for i in range(4100)]
    codes, params, table = cache(lens[:64], 1, 16, 64, seed=3)
    table = table[[i % 64 for i in range(4100)]].contiguous()
    lens = [lens[i % 64] for i in range(4100)]
    q = torch.randn(4100, 128, device=DEV).bfloat16()
    o = B.attention_decode_kv4(q, codes, params, table, torch.tensor(lens, dtype=torch.int32, device=DEV), 2)
    pick = [0, 1, 63, 4095, 4096, 4099]
    want, bound = decode_reference(q[pick], codes, params, table[pick], [lens[i] for i in pick], 2)
    assert bool(((o[pick].double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype,shape", [(torch.bfloat16, (3, 2, 9, 4, 16, 64)), (torch.float32, (1, 2, 9, 3, 5, 48)),
                                         (torch.uint8, (2, 2, 9, 2, 7, 24)), (torch.uint8, (9, 1, 3, 5)),
                                         (torch.bfloat16, (2, 2, 9, 3, 7, 2)), (torch.bfloat16, (2, 2, 9, 8, 64, 128))])
def test_copy_pages(dtype, shape):
    g = torch.Generator(device=DEV).manual_seed(0)
    pool = torch.randint(0, 200, shape, generator=g, device=DEV).to(dtype)
    n_pages, page = shape[-4], shape[-2]
    want = pool.clone()
    src, dst = [1, 7, 1], [0, 3, 8]
    v, w = pool.view(-1, *shape[-4:]), want.view(-1, *shape[-4:])
    for s, d in zip(src, dst):
        w[:, d] = v[:, s]
    B.copy_pages(pool, src, dst)
    assert torch.equal(pool, want)
    rows = [2, 0, page]
    src, dst = [2, 4, 5], [6, 0, 3]
    for s, d, r in zip(src, dst, rows):
        w[:, d, :, :r] = w[:, s, :, :r].clone()
    as_t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    B.copy_pages(pool, as_t(src), as_t(dst), rows=as_t(rows))
    assert torch.equal(pool, want)
    B.copy_pages(pool, [], [])
    B.copy_pages(pool, as_t([5, -1, n_pages]), as_t([5, 0, 1]))   # itself; two pages that do not exist
    with pytest.raises(B.B200Error):
        B.device_status()
    assert torch.equal(pool, want)


def test_copy_pages_refusals():
    pool = torch.zeros(2, 2, 6, 2, 16, 64, device=DEV).bfloat16()
    t = torch.zeros(2, dtype=torch.int32, device=DEV)
    for call, status in [(lambda: B.copy_pages(pool, [0], [6]), 1), (lambda: B.copy_pages(pool, [0, 1], [2, 2]), 1),
                         (lambda: B.copy_pages(pool, [0, 1], [1, 2]), 1), (lambda: B.copy_pages(pool, [0], [1, 2]), 2),
                         (lambda: B.copy_pages(pool, t, [1, 2]), 1), (lambda: B.copy_pages(pool, t, t.long()), 3),
                         (lambda: B.copy_pages(pool[:, :, ::2], [0], [1]), 2), (lambda: B.copy_pages(pool.cpu(), [0], [1]), 1),
                         (lambda: B.compact_pages(pool, t, t, t.view(1, 2), t), 2),
                         (lambda: B.compact_pages(pool, t, t, t.view(1, 2).long(), t), 3)]:
        with pytest.raises(B.B200Error) as e:
            call()
        assert e.value.status == status


def test_decode_refusals():
    codes, params, table = cache([40], 2, 16, 64)
    q = torch.randn(1, 256, device=DEV).bfloat16()
    ctx = torch.tensor([40], dtype=torch.int32, device=DEV)
    for call, status in [
        (lambda: B.attention_decode_kv4(q, codes, params, table, ctx, 3), 2),
        (lambda: B.attention_decode_kv4(q.half(), codes, params, table, ctx, 4), 3),
        (lambda: B.attention_decode_kv4(q, codes, params, table, ctx.long(), 4), 3),
        (lambda: B.attention_decode_kv4(q, codes, params[:1], table, ctx, 4), 2),
        (lambda: B.attention_decode_kv4(q, codes[0], params, table, ctx, 4), 2),
        (lambda: B.attention_decode_kv4(q, codes, params, table.expand(2, -1), ctx, 4), 3),
        (lambda: B.attention_decode_kv4(q, codes, params, table, ctx, 4, scratch=torch.empty(64, dtype=torch.uint8, device=DEV)), 5),
        (lambda: B.attention_decode_kv4(q.float(), codes, params, table, ctx, 4, impl=1), 10),
        (lambda: B.attention_decode_kv4(q, codes, params, table, ctx, 4, impl=7), 1),
        (lambda: B.kv4_append(q, q, codes, params, table, cu_of([1])), 2),
        (lambda: B.kv4_append(q[:, :128].half(), q[:, :128].half(), codes, params, table, cu_of([1])), 3),
        (lambda: B.kv4_append(q[:, :128], q[:, :128], codes, params, table, cu_of([1, 1])), 2),
    ]:
        with pytest.raises(B.B200Error) as e:
            call()
        assert e.value.status == status


@pytest.mark.parametrize("hs,heads,hk,page", [(128, 8, 2, 64), (64, 4, 4, 16)])
def test_serving_run(hs, heads, hk, page):
    """Prompts through packed attention, their keys and values into a 4-bit cache, two continuations of one prompt that
    share its pages, decode steps, one continuation ends, the pool is compacted, decoding goes on unchanged."""
    g = torch.Generator(device=DEV).manual_seed(3)
    lens = [page * 2 + 5, 3, page]
    L, n_pages = 2, 24
    alloc = B.PageAllocator(n_pages)
    codes, params = B.new_kv4_pages(L, n_pages, hk, page, hs)
    width = 5
    seqs = [alloc.alloc(-(-(n + 2) // page)) for n in lens]
    as_table = lambda seqs: torch.tensor([s + [-1] * (width - len(s)) for s in seqs], dtype=torch.int32, device=DEV)
    cu = cu_of(lens)
    for l in range(L):
        qkv = torch.randn(sum(lens), (heads + 2 * hk) * hs, generator=g, device=DEV).bfloat16()
        q, k, v = qkv[:, :heads * hs], qkv[:, heads * hs:(heads + hk) * hs], qkv[:, (heads + hk) * hs:]
        o, _ = B.attention_packed(q, k, v, cu, heads, hk)
        B.kv4_append(k, v, codes[l], params[l], as_table(seqs), cu)
        # the prompts' last rows attend to the same keys a decode step over the cache sees, up to the 4 bits
        last = cu[1:].long() - 1
        ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
        od = B.attention_decode_kv4(q[last].contiguous(), codes[l], params[l], as_table(seqs), ctx, heads)
        rk, rv = B.kv4_read(codes[l], params[l], as_table(seqs), cu, None, sum(lens))
        oq, _ = B.attention_packed(q, rk, rv, cu, heads, hk)
        # rk, rv are rounded to bf16 once more: scores move by U sum|q||k| / sqrt(hs) <= U |q||k| / sqrt(hs) = U S, weights
        # by twice that, values by U; both kernels round weights and outputs: together U max|v| (2 S + 1 + 2 + 2)
        S = float(q.float().view(-1, hs).norm(dim=1).max() * rk.float().view(-1, hs).norm(dim=1).max()) / math.sqrt(hs)
        tol = 2.0 ** -8 * float(rv.float().abs().max()) * (2 * S + 5)
        assert float((od.float() - oq[last].float()).abs().max()) < tol
    # sequence 0 forks: full pages shared, the partly filled one copied
    child, copies = alloc.fork(seqs[0], lens[0], page)
    for pool in (codes, params):
        B.copy_pages(pool, [c[0] for c in copies], [c[1] for c in copies], rows=[c[2] for c in copies])
    seqs.append(child)
    lens = lens + [lens[0]]
    table = as_table(seqs)
    step = torch.randn(4, 2 * hk * hs, generator=g, device=DEV).bfloat16()
    one = torch.arange(5, dtype=torch.int32, device=DEV)
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    for l in range(L):
        B.kv4_append(step[:, :hk * hs], step[:, hk * hs:], codes[l], params[l], table, one, ctx)
    ctx += 1
    q = torch.randn(4, heads * hs, generator=g, device=DEV).bfloat16()
    outs = [B.attention_decode_kv4(q, codes[l], params[l], table, ctx, heads) for l in range(L)]
    for l in range(L):   # parent and child differ only in their newest row
        want, bound = decode_reference(q, codes[l], params[l], table, [n + 1 for n in lens], heads)
        assert bool(((outs[l].double() - want).abs() <= bound).all())
    alloc.free(seqs[1])
    alloc.free(seqs[0])          # the child keeps the shared pages
    keep = [2, 3]
    table = as_table([seqs[i] for i in keep])
    src, dst, page_map = alloc.compact()
    assert src and max(dst) < n_pages - alloc.free_pages
    B.compact_pages([codes, params], src, dst, table, page_map)
    assert table.tolist() == as_table([[page_map[p] for p in seqs[i]] for i in keep]).tolist()
    for l in range(L):
        again = B.attention_decode_kv4(q[keep], codes[l], params[l], table, ctx[keep], heads)
        want, bound = decode_reference(q[keep], codes[l], params[l], table, [lens[i] + 1 for i in keep], heads)
        assert bool(((again.double() - want).abs() <= bound).all())
    alloc.free([page_map[p] for p in seqs[2]])
    alloc.free([page_map[p] for p in seqs[3]])
    assert alloc.free_pages == n_pages
    assert B.device_status() == 0


def test_two_graphs_and_streams():
    """Two captured decode steps over one cache, replayed on two streams at once, and an eager call beside them."""
    lens, heads, hk, hs, page = [900, 30], 8, 2, 128, 64
    codes, params, table = cache(lens, hk, page, hs, seed=1)
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    qs = [torch.randn(2, heads * hs, device=DEV).bfloat16() for _ in range(3)]
    want = [B.attention_decode_kv4(q, codes, params, table, ctx, heads) for q in qs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q in qs[:2]:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(B.attention_decode_kv4(q, codes, params, table, ctx, heads))
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        eager = B.attention_decode_kv4(qs[2], codes, params, table, ctx, heads)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs + [eager], want))
