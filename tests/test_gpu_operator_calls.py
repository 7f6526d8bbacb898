"""Calls of the packed, 4-bit and page operators at the edges of what their documentation allows."""
import math

import pytest
import torch

import b200_llama as B

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
