"""Decode attention over the 4-bit cache where the weights of a head are far from equal: one key that carries most of the
weight over a long tail that carries the rest, scores spread over many powers of e, value rows of very different scales,
and rows that read back as NaN."""
import math

import pytest
import torch

import b200_llama as B

pytestmark = pytest.mark.gpu
DEV = "cuda"
U32 = 2.0 ** -24
U = {torch.float32: U32, torch.bfloat16: 2.0 ** -8}
TILE = 32   # keys whose weights share a step


def pages_of(batch, n, page, seed):
    width = -(-n // page)
    perm = torch.randperm(batch * width, generator=torch.Generator().manual_seed(seed))
    return perm.view(batch, width).int().to(DEV), batch * width


def pool_of(k, v, table, page):
    """Pools from rows given as (codes [batch, n, hk, hs] 0..15, scale, minimum [batch, n, hk])."""
    batch, n, hk, hs = k[0].shape
    width = table.shape[1]
    codes = torch.zeros(2, batch * width, hk, page, hs // 2, dtype=torch.uint8, device=DEV)
    params = torch.full((2, batch * width, hk, page, 2), math.nan, device=DEV).bfloat16()
    at = torch.arange(n, device=DEV)
    pg, r = table.long()[:, at // page], (at % page).expand(batch, n)
    for half, (c, sc, lo) in enumerate((k, v)):
        codes[half, pg, :, r] = c[..., 0::2] | (c[..., 1::2] << 4)
        params[half, pg, :, r] = torch.stack((sc, lo), -1).bfloat16()
    return codes, params


def reference(q, k, v, heads, impl_tc):
    """Output of one sequence in 64 bits and the bound of a kernel: rows as (codes [n, hk, hs], scale, minimum [n, hk]),
    q [heads * hs].  With U half a step of a type,
      ds <= (hs + 16) U32 sum|q| (|lo| + 15 sc) / sqrt(hs) + 16 U32 |s|           fp32 sums of a score
            + 1.01 max|q| / 65024 sum(code) sc / sqrt(hs)                         the query in steps of 1/32512 (tensor cores)
      |do| <= U|o| + 2 max(ds) sum p|v| + (n + 48) U32 sum p (|lo| + 15 sc)
            + sum over tiles of 32 keys: max(p sc) / 65535 sum(code)              weights p sc in steps of 2^(e+1)/65535, 2^e
                                                                                  the power of two of the tile's largest (tensor cores)
    Nothing in it grows with the number of keys times the largest weight."""
    n, hk, hs = k[0].shape
    group = heads // hk
    small = q.dtype == torch.bfloat16
    out = torch.zeros(heads, hs, dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(out)
    Q = q.view(heads, hs).double()
    for j in range(hk):
        kc, ks, kl = k[0][:, j].double(), k[1][:, j, None].double(), k[2][:, j, None].double()
        vc, vs, vl = v[0][:, j].double(), v[1][:, j, None].double(), v[2][:, j, None].double()
        K, V = kl + ks * kc, vl + vs * vc
        for h in range(j * group, (j + 1) * group):
            s = K @ Q[h] / math.sqrt(hs)
            p = torch.softmax(s, 0)
            ds = (hs + 16) * U32 * Q[h].abs().sum() * (15 * ks + kl.abs())[:, 0] / math.sqrt(hs) + 16 * U32 * s.abs()
            if impl_tc:
                ds = ds + 1.01 * Q[h].abs().max() / 65024 * kc.sum(1) * ks[:, 0] / math.sqrt(hs)
            out[h] = p @ V
            bound[h] = U[q.dtype] * out[h].abs() + 2 * ds.max() * (p @ V.abs()) + (n + 48) * U32 * (p @ (15 * vs + vl.abs()))
            if impl_tc:
                pad = -n % TILE
                w = torch.nn.functional.pad(p * vs[:, 0], (0, pad)).view(-1, TILE).amax(1)
                c = torch.nn.functional.pad(vc, (0, 0, 0, pad)).view(-1, TILE, hs).sum(1)
                bound[h] += (w / 65535) @ c
    assert small or not impl_tc
    return out.view(-1), bound.view(-1) + 1e-30


def bf16(x):
    return x.bfloat16().float()


def rows(g, batch, n, hk, hs, low, high, shift):
    """Random rows: scales in low .. high, values centred `shift` scales away from zero."""
    c = torch.randint(0, 16, (batch, n, hk, hs), generator=g, device=DEV, dtype=torch.uint8)
    sc = bf16(low + (high - low) * torch.rand(batch, n, hk, generator=g, device=DEV))
    return c, sc, bf16((shift - 7.5) * sc)


def queries(g, batch, heads, hk, hs):
    """Heads of a group agree in their elements' signs, so that one key can stand out for all of them."""
    sign = torch.randint(0, 2, (batch, hk, 1, hs), generator=g, device=DEV).float() * 2 - 1
    size = torch.rand(batch, hk, heads // hk, hs, generator=g, device=DEV) + 0.5
    return (sign * size).view(batch, heads * hs).bfloat16(), sign[:, :, 0]


def check(q, k, v, table, page, n, heads, impl, pick=None):
    codes, params = pool_of(k, v, table, page)
    batch = q.shape[0]
    ctx = torch.full((batch,), n, dtype=torch.int32, device=DEV)
    o = B.attention_decode_kv4(q, codes, params, table, ctx, heads, impl=impl)
    assert B.device_status() == 0
    for b in range(batch) if pick is None else pick:
        want, bound = reference(q[b], [x[b] for x in k], [x[b] for x in v], heads, impl == 0 and q.dtype == torch.bfloat16)
        err = (o[b].double() - want).abs()
        assert bool((err <= bound).all()), (b, float((err / bound).max()))
    return o


def stand_out(k, sign, at, gap):
    """Key `at` of every head points along the queries, its score about `gap` above zero."""
    hs = k[0].shape[-1]
    for b in range(k[0].shape[0]):
        k[0][b, at[b]] = torch.where(sign[b] > 0, 15, 0).to(torch.uint8)
        k[1][b, at[b]] = bf16(torch.tensor(gap / (7.5 * math.sqrt(hs)), device=DEV))
        k[2][b, at[b]] = bf16(-7.5 * k[1][b, at[b]])


@pytest.mark.parametrize("impl", [0, 2])
@pytest.mark.parametrize("share", [0.5, 0.9, 0.99])
@pytest.mark.parametrize("n,heads,hk,hs,page", [(250, 8, 2, 128, 64), (1024, 4, 2, 64, 16), (4096, 8, 2, 128, 64),
                                                (4096, 16, 2, 64, 128), (32768, 2, 2, 128, 64)])
def test_one_key_carries_most_of_the_weight(n, heads, hk, hs, page, share, impl):
    """The key is the first, the second, one of another warp, the last; its value row is small in the first key head and
    like the others in the second.  The values are off centre, so that a row read as its minimum would show."""
    g = torch.Generator(device=DEV).manual_seed(n + hs)
    at = [0, 1, 33, n - 1]
    k, v = rows(g, 4, n, hk, hs, 0.02, 0.06, 0.0), rows(g, 4, n, hk, hs, 0.05, 0.35, 3.0)
    q, sign = queries(g, 4, heads, hk, hs)
    stand_out(k, sign, at, math.log(n * share / (1 - share)))
    for b in range(4):
        v[1][b, at[b], 0] = bf16(0.05 * v[1][b, at[b], 0])
        v[2][b, at[b], 0] = bf16(-7.5 * v[1][b, at[b], 0])
    table, _ = pages_of(4, n, page, seed=n)
    check(q, k, v, table, page, n, heads, impl)


def test_the_same_with_whole_segments_in_a_cta():
    g = torch.Generator(device=DEV).manual_seed(3)
    batch, n, hk, hs, page = 80, 512, 8, 128, 64
    k, v = rows(g, batch, n, hk, hs, 0.02, 0.06, 0.0), rows(g, batch, n, hk, hs, 0.05, 0.35, 3.0)
    q, sign = queries(g, batch, hk, hk, hs)
    stand_out(k, sign, [(7 * b) % n for b in range(batch)], math.log(n * 20))
    table, _ = pages_of(batch, n, page, seed=1)
    check(q, k, v, table, page, n, hk, 0, pick=[0, 1, 31, 40, 79])


@pytest.mark.parametrize("impl", [0, 2])
@pytest.mark.parametrize("n,heads,hk,hs", [(300, 4, 1, 128), (4096, 8, 1, 64), (4096, 4, 2, 128)])
def test_scores_over_many_powers(n, heads, hk, hs, impl):
    """Random scores of a spread of 5: the largest weight changes from tile to tile, upwards and downwards."""
    g = torch.Generator(device=DEV).manual_seed(n)
    k, v = rows(g, 2, n, hk, hs, 0.8, 1.2, 0.0), rows(g, 2, n, hk, hs, 0.05, 0.35, 3.0)
    q, _ = queries(g, 2, heads, hk, hs)
    table, _ = pages_of(2, n, 64, seed=n)
    check(q, k, v, table, 64, n, heads, impl)


@pytest.mark.parametrize("impl", [0, 2])
@pytest.mark.parametrize("factor", [1e3, 1e6, 1e30])
def test_a_value_row_of_another_size(factor, impl):
    """One value row far larger than the others whose key is not seen (a score of -80), one far smaller than the others
    that is: neither decides how exactly the others are read."""
    g = torch.Generator(device=DEV).manual_seed(5)
    n, heads, hk, hs, page = 2000, 4, 2, 128, 64
    k, v = rows(g, 2, n, hk, hs, 0.02, 0.06, 0.0), rows(g, 2, n, hk, hs, 0.05, 0.35, 3.0)
    q, sign = queries(g, 2, heads, hk, hs)
    stand_out(k, -sign, [0, 40], 80.0 + math.log(factor))
    for b, at in enumerate((0, 40)):
        v[1][b, at], v[2][b, at] = bf16(v[1][b, at] * factor), bf16(v[2][b, at] * factor)
        v[1][b, at + 5], v[2][b, at + 5] = bf16(v[1][b, at + 5] / factor), bf16(v[2][b, at + 5] / factor)
    # the score falls with the logarithm of the factor: what the large row still adds is below any other weight
    table, _ = pages_of(2, n, page, seed=2)
    check(q, k, v, table, page, n, heads, impl)


@pytest.mark.parametrize("impl", [0, 2])
@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("half", [0, 1])
def test_rows_that_read_back_as_nan(hs, half, impl):
    """A row that held an infinity when it was appended reads back as NaN: the heads that see it come out NaN, the other
    heads, sequences and rows behind the end do not."""
    g = torch.Generator(device=DEV).manual_seed(7)
    n, heads, hk, page = 600, 4, 2, 64
    k, v = rows(g, 3, n, hk, hs, 0.02, 0.2, 0.0), rows(g, 3, n, hk, hs, 0.05, 0.35, 0.0)
    q, _ = queries(g, 3, heads, hk, hs)
    table, _ = pages_of(3, n, page, seed=3)
    codes, params = pool_of(k, v, table, page)
    params[half, int(table[1, 400 // page]), 0, 400 % page] = math.nan   # sequence 1, key head 0
    params[half, int(table[2, 500 // page]), 1, 500 % page] = math.nan   # sequence 2: behind its end
    lens = [n, n, 500]
    o = B.attention_decode_kv4(q, codes, params, table, torch.tensor(lens, dtype=torch.int32, device=DEV), heads, impl=impl)
    assert B.device_status() == 0
    o3 = o.view(3, hk, -1)
    assert bool(o3[1, 0].isnan().all())
    for b in range(3):
        want, bound = reference(q[b], [x[b, :lens[b]] for x in k], [x[b, :lens[b]] for x in v], heads, impl == 0)
        ok = ((o[b].double() - want).abs() <= bound).view(hk, -1)
        assert bool(ok[1].all()) and (b == 1 or bool(ok[0].all()))


@pytest.mark.parametrize("heads,hk,hs,dtype,impl", [(4, 2, 64, torch.bfloat16, 0), (4, 2, 128, torch.bfloat16, 0),
                                                    (4, 2, 64, torch.bfloat16, 2), (6, 3, 48, torch.float32, 0)])
@pytest.mark.parametrize("dead", [32, 192, 384])   # whole tiles
def test_scores_of_minus_infinity(heads, hk, hs, dtype, impl, dead):
    """Keys of the type's lowest value, whose scores overflow to minus infinity, have no weight, however many come first."""
    g = torch.Generator(device=DEV).manual_seed(9)
    n, page = 400, 16
    k, v = rows(g, 2, n, hk, hs, 0.02, 0.2, 0.0), rows(g, 2, n, hk, hs, 0.05, 0.35, 1.0)
    q = (torch.rand(2, heads * hs, generator=g, device=DEV) + 0.5).to(dtype)
    k[1][:, :dead], k[2][:, :dead] = 0.0, bf16(torch.tensor(torch.finfo(torch.bfloat16).min, device=DEV))
    table, _ = pages_of(2, n, page, seed=9)
    codes, params = pool_of(k, v, table, page)
    o = B.attention_decode_kv4(q, codes, params, table, torch.tensor([n, dead], dtype=torch.int32, device=DEV), heads, impl=impl)
    assert B.device_status() == 0
    want, bound = reference(q[0], [x[0, dead:] for x in k], [x[0, dead:] for x in v], heads, impl == 0 and dtype == torch.bfloat16)
    assert bool(((o[0].double() - want).abs() <= bound).all())
    assert bool((o[1] == 0).all())


@pytest.mark.parametrize("heads,hk,hs,dtype,impl", [(4, 2, 64, torch.bfloat16, 0), (4, 2, 128, torch.bfloat16, 2),
                                                    (6, 3, 48, torch.float32, 0)])
@pytest.mark.parametrize("half", [0, 1])
def test_first_rows_that_read_back_as_nan(heads, hk, hs, dtype, half, impl):
    """The rows a lane meets first are NaN, before it has any number to compare with."""
    g = torch.Generator(device=DEV).manual_seed(11)
    n, page = 300, 16
    k, v = rows(g, 2, n, hk, hs, 0.02, 0.2, 0.0), rows(g, 2, n, hk, hs, 0.05, 0.35, 1.0)
    q, _ = queries(g, 2, heads, hk, hs)
    table, _ = pages_of(2, n, page, seed=9)
    codes, params = pool_of(k, v, table, page)
    for pg in table[0, :9].tolist():
        params[half, pg, 0] = math.nan        # 144 rows of sequence 0, key head 0
    o = B.attention_decode_kv4(q.to(dtype), codes, params, table, torch.tensor([n, n], dtype=torch.int32, device=DEV), heads, impl=impl)
    assert B.device_status() == 0
    bad = o.view(2, hk, -1).isnan()
    assert bool(bad[0, 0].all()) and not bool(bad[0, 1:].any()) and not bool(bad[1].any())
