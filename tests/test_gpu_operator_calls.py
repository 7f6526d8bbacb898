"""Calls of the packed, 4-bit and page operators at the edges of what their documentation allows."""
import math

import pytest
import torch

import b200_llama as B
import packed_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("order", [(0, 1), (1, 0), (1,)])
def test_compact_with_a_pool_that_holds_nothing(order):
    full = torch.arange(6, device=DEV).float().view(1, 6, 1, 1, 1).expand(2, 6, 2, 4, 8).contiguous()
    empty = torch.zeros(0, 6, 2, 4, 8, device=DEV)
    table = torch.tensor([[5, 4, 2, -1]], dtype=torch.int32, device=DEV)
    B.compact_pages([(full, empty)[i] for i in order], [5, 4], [0, 1], table, [0, 1, 2, 3, 1, 0])
    assert B.device_status() == 0 and table.tolist() == [[0, 1, 2, -1]]
    if 0 in order:
        assert full[0, :, 0, 0, 0].tolist() == [5, 4, 2, 3, 4, 5]


@pytest.mark.parametrize("batch,heads,hk,hs,dtype", [(3, 4, 2, 64, torch.bfloat16), (700, 32, 8, 128, torch.bfloat16),
                                                     (2, 6, 6, 48, torch.float32)])
@pytest.mark.parametrize("n_pages", [0, 2])
def test_page_tables_without_columns(batch, heads, hk, hs, dtype, n_pages):
    """A cache that holds nothing yet: every sequence has zero rows and gets zeros; appended rows have no place."""
    codes, params = B.new_kv4_pages(1, n_pages, hk, 16, hs)
    table = torch.zeros(batch, 0, dtype=torch.int32, device=DEV)
    ctx = torch.zeros(batch, dtype=torch.int32, device=DEV)
    q = torch.randn(batch, heads * hs, device=DEV).to(dtype)
    o = B.attention_decode_kv4(q, codes[0], params[0], table, ctx, heads, out=torch.full_like(q, 7.0))
    assert B.device_status() == 0 and bool((o == 0).all())
    none = torch.zeros(batch + 1, dtype=torch.int32, device=DEV)
    kv = torch.randn(2, hk * hs, device=DEV).to(dtype)
    B.kv4_append(kv, kv, codes[0], params[0], table, none)
    assert B.device_status() == 0
    none[-1] = 2
    B.kv4_append(kv, kv, codes[0], params[0], table, none)
    with pytest.raises(B.B200Error) as e:
        B.device_status()
    assert e.value.status == 1 and bool((params == 0).all())
    # a pool without pages under tables that name some: skipped and reported
    if n_pages == 0:
        table = torch.zeros(batch, 1, dtype=torch.int32, device=DEV)
        o = B.attention_decode_kv4(q, codes[0], params[0], table, ctx + 3, heads, out=torch.full_like(q, 7.0))
        with pytest.raises(B.B200Error) as e:
            B.device_status()
        assert e.value.status == 1 and bool((o == 0).all())


@pytest.mark.parametrize("impl", [0, 2])
@pytest.mark.parametrize("hs,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (48, torch.float32)])
@pytest.mark.parametrize("what", ["q", "k"])
def test_a_nan_in_the_first_key_or_a_query(what, hs, dtype, impl):
    """A score that is NaN makes its row NaN, also where it is the first one the row meets; other sequences are untouched."""
    g = torch.Generator(device=DEV).manual_seed(0)
    lens, heads, kv = [30, 200, 170], 4, 2
    q, k, v = (torch.randn(400, n * hs, generator=g, device=DEV).to(dtype) for n in (heads, kv, kv))
    cu = torch.tensor([0, 30, 230, 400], dtype=torch.int32, device=DEV)
    clean, clean_lse = B.attention_packed(q, k, v, cu, heads, kv, impl=impl)
    if what == "k":
        k[30, 3] = math.nan                       # key head 0: query heads 0 and 1 of the second sequence
        rows, cols = slice(30, 230), slice(0, 2 * hs)
    else:
        q[130, 3] = math.nan                      # query head 0
        rows, cols = slice(130, 131), slice(0, hs)
    o, lse = B.attention_packed(q, k, v, cu, heads, kv, impl=impl)
    assert B.device_status() == 0
    bad = torch.zeros_like(o, dtype=torch.bool)
    bad[rows, cols] = True
    assert torch.equal(o.isnan(), bad) and torch.equal(o[~bad], clean[~bad])
    bad_lse = torch.zeros_like(lse, dtype=torch.bool)
    bad_lse[:cols.stop // hs, rows] = True
    assert torch.equal(lse.isnan(), bad_lse) and torch.equal(lse[~bad_lse], clean_lse[~bad_lse])


@pytest.mark.parametrize("heads,kv,hs", [(4, 2, 64), (4, 1, 128), (3, 3, 128)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_whole_sequences_that_are_not_finite(heads, kv, hs, bad):
    """Every other sequence of a batch holds nothing but infinities or NaN, in every operand; many of them share tiles.  The
    others come out as if they were alone, forward and backward, and to the bit again."""
    g = torch.Generator(device=DEV).manual_seed(1)
    lens = [5, 30, 1, 60, 100, 3, 1, 1, 250, 7, 129, 64, 2, 40]
    T, cu = sum(lens), torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    q, k, v, d_o = (torch.randn(T, n * hs, generator=g, device=DEV).bfloat16() for n in (heads, kv, kv, heads))
    ro, rl, bo, bl = R.forward(q, k, v, lens, heads, kv)
    want, bounds = R.backward(q, k, v, d_o, lens, heads, kv)
    fine = torch.ones(T, dtype=torch.bool, device=DEV)
    for i in range(0, len(lens), 2):
        fine[cu[i]:cu[i + 1]] = False
    for x in (q, k, v, d_o):
        x[~fine] = bad
    first = None
    for _ in range(2):
        o, lse = B.attention_packed(q, k, v, cu, heads, kv)
        grads = B.attention_packed_backward(q, k, v, o, lse, d_o, cu, heads, kv)
        assert B.device_status() == 0
        assert bool(((o.double() - ro).abs() <= bo)[fine].all()) and not bool(o[~fine].isfinite().any())
        assert bool(((lse.double() - rl).abs() <= bl)[:, fine].all())
        for x, r, b in zip(grads, want, bounds):
            assert bool(((x.double() - r).abs() <= b)[fine].all())
        if first is not None:
            assert all(torch.equal(x[fine], y[fine]) for x, y in zip((o,) + grads, first))
        first = (o,) + grads


@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_one_row_that_is_not_finite_in_each_operand(bad):
    """Rows after and before it, in its own tile and in others: what does not see it is as it was, what sees it is not finite."""
    T, heads, kv, hs = 600, 4, 2, 128
    g = torch.Generator(device=DEV).manual_seed(2)
    cu = torch.tensor([0, T], dtype=torch.int32, device=DEV)
    ops = [torch.randn(T, n * hs, generator=g, device=DEV).bfloat16() for n in (heads, kv, kv, heads)]
    o, lse = B.attention_packed(*ops[:3], cu, heads, kv)
    clean = B.attention_packed_backward(*ops[:3], o, lse, ops[3], cu, heads, kv)
    want, bounds = R.backward(*ops, [T], heads, kv)
    ro, _, bo, _ = R.forward(*ops[:3], [T], heads, kv)
    at = 300
    for i in range(4):
        x = [t.clone() for t in ops]
        x[i][at, 5] = bad                                        # key or query head 0
        oo, ll = B.attention_packed(*x[:3], cu, heads, kv)
        dq, dk, dv = B.attention_packed_backward(*x[:3], o, lse, x[3], cu, heads, kv)
        assert B.device_status() == 0
        if i in (1, 2):                                          # a key or value row: rows before it do not see it
            assert bool(((oo.double() - ro).abs() <= bo)[:at].all())
            seen = ops[0][at:, 5] > 0 if i == 1 and bad == math.inf else slice(None)   # q < 0: a score of minus infinity, no weight
            assert not bool(oo[at:, 5][seen].isfinite().any())
            assert bool(((dq.double() - want[0]).abs() <= bounds[0])[:at].all())
        else:                                                    # a query or cotangent row: later keys are not seen by it
            for y, r, b in zip((dk, dv), want[1:], bounds[1:]):
                assert bool(((y.double() - r).abs() <= b)[at + 1:].all())
            rest = torch.arange(T, device=DEV) != at
            assert bool(((dq.double() - want[0]).abs() <= bounds[0])[rest].all()) and not bool(dq[at, :hs].isfinite().any())
        other = slice(hs, kv * hs)                               # the second key head
        assert torch.equal(dk[:, other], clean[1][:, other]) and torch.equal(dv[:, other], clean[2][:, other])


@pytest.mark.parametrize("what", ["k", "v"])
def test_a_nan_does_not_cost_a_pass_over_every_row(what):
    """One NaN in an early row, which every later row sees: they are NaN by right, and nothing is computed again for them.
    (A pass pair by pair takes 600 to 1400 times as long as the products.)"""
    T, heads, kv, hs = 4096, 8, 2, 128
    g = torch.Generator(device=DEV).manual_seed(0)
    q, k, v, d_o = (torch.randn(T, n * hs, generator=g, device=DEV).bfloat16() for n in (heads, kv, kv, heads))
    cu = torch.tensor([0, T], dtype=torch.int32, device=DEV)

    def passes():
        o, lse = B.attention_packed(q, k, v, cu, heads, kv)
        return (lambda: B.attention_packed(q, k, v, cu, heads, kv),
                lambda: B.attention_packed_backward(q, k, v, o, lse, d_o, cu, heads, kv))

    def time(f):
        best = math.inf
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            f()
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    before = [time(f) for f in passes()]
    (k if what == "k" else v)[T // 4, 3] = math.nan
    after = [time(f) for f in passes()]
    assert all(a < 30 * b for a, b in zip(after, before)), (before, after)
