"""Packed causal attention with grouped heads, forward and backward, against 64-bit formulas with derived bounds."""
import math

import pytest
import torch

import b200_llama as B
import packed_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def cu_of(lens, gap=0):
    cu = [gap]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device=DEV)


def make(lens, heads, kv_heads, hs, dtype, seed=0, gap=0, tail=0, gain=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    T = gap + sum(lens) + tail
    qkv = (torch.randn(T, (heads + 2 * kv_heads) * hs, generator=g, device=DEV) * gain).to(dtype)
    d_o = torch.randn(T, heads * hs, generator=g, device=DEV).to(dtype)
    return qkv[:, :heads * hs], qkv[:, heads * hs:(heads + kv_heads) * hs], qkv[:, (heads + kv_heads) * hs:], d_o


def check_fwd(q, k, v, lens, heads, kv_heads, impl=0, gap=0):
    o, lse = B.attention_packed(q, k, v, cu_of(lens, gap), heads, kv_heads, impl=impl)
    assert B.device_status() == 0
    ro, rl, bo, bl = R.forward(q, k, v, lens, heads, kv_heads, gap)
    live = ~ro.isnan()
    assert bool(((o.double() - ro).abs() <= bo)[live].all()), float(((o.double() - ro).abs() / bo)[live].max())
    live = ~rl.isnan()
    assert bool(((lse.double() - rl).abs() <= bl)[live].all()), float(((lse.double() - rl).abs() / bl)[live].max())
    return o, lse


SHAPES = [  # lens, heads, kv_heads, hs, dtype
    ([1], 6, 6, 48, torch.float32),
    ([17, 1, 5], 6, 2, 48, torch.float32),
    ([0, 3, 0, 0, 40, 0], 2, 1, 16, torch.float32),
    ([33, 64, 31], 4, 4, 32, torch.bfloat16),
    ([100, 257], 4, 2, 64, torch.float32),
    ([1], 2, 1, 64, torch.bfloat16),
    ([1] * 200, 4, 2, 64, torch.bfloat16),
    ([128], 2, 2, 64, torch.bfloat16),
    ([129, 127, 1, 255], 4, 1, 64, torch.bfloat16),
    ([0, 300, 0, 5, 700, 1], 6, 2, 64, torch.bfloat16),
    ([1], 4, 1, 128, torch.bfloat16),
    ([127, 2, 128, 640], 4, 2, 128, torch.bfloat16),
    ([3] * 70 + [500], 8, 2, 128, torch.bfloat16),
    ([1000, 24], 3, 1, 128, torch.bfloat16),
    ([250, 90], 2, 2, 128, torch.float32),
]


@pytest.mark.parametrize("impl", [0, 2])
@pytest.mark.parametrize("lens,heads,kv_heads,hs,dtype", SHAPES)
def test_forward(lens, heads, kv_heads, hs, dtype, impl):
    q, k, v, _ = make(lens, heads, kv_heads, hs, dtype, seed=len(lens))
    check_fwd(q, k, v, lens, heads, kv_heads, impl)


@pytest.mark.parametrize("impl", [0, 2])
@pytest.mark.parametrize("lens,heads,kv_heads,hs,dtype", SHAPES)
def test_backward(lens, heads, kv_heads, hs, dtype, impl):
    q, k, v, d_o = make(lens, heads, kv_heads, hs, dtype, seed=3 + len(lens))
    cu = cu_of(lens)
    o, lse = B.attention_packed(q, k, v, cu, heads, kv_heads, impl=impl)
    got = B.attention_packed_backward(q, k, v, o, lse, d_o, cu, heads, kv_heads, impl=impl)
    assert B.device_status() == 0
    want, bounds = R.backward(q, k, v, d_o, lens, heads, kv_heads)
    for name, x, r, b in zip(("dq", "dk", "dv"), got, want, bounds):
        err = (x.double() - r).abs()
        assert bool((err <= b).all()), (name, float((err / b).max()))


@pytest.mark.parametrize("hs,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (48, torch.float32)])
@pytest.mark.parametrize("gain", [3.0, 8.0])
def test_forward_wide_scores(hs, dtype, gain):
    """Scores spread over hundreds: the running maximum of a row is raised many times."""
    lens = [700, 13, 300]
    q, k, v, _ = make(lens, 4, 2, hs, dtype, seed=9, gain=gain)
    check_fwd(q, k, v, lens, 4, 2)


@pytest.mark.parametrize("impl", [0, 2])
@pytest.mark.parametrize("hs,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (32, torch.float32)])
def test_rows_of_no_sequence(hs, dtype, impl):
    """Rows before the first and behind the last sequence hold NaN and infinities: nothing of them arrives anywhere, and
    the outputs there stay as they were."""
    lens, gap, tail, heads, kv = [70, 1, 200], 5, 40, 4, 2
    q, k, v, d_o = make(lens, heads, kv, hs, dtype, seed=4, gap=gap, tail=tail)
    end = gap + sum(lens)
    clean = [t.clone() for t in (q, k, v, d_o)]
    for t in (q, k, v, d_o):
        t[:gap] = math.nan
        t[end:end + 20] = math.inf
        t[end + 20:] = math.nan
    T, cu = q.shape[0], cu_of(lens, gap)
    out = torch.full((T, heads * hs), 7.0, dtype=dtype, device=DEV)
    lse = torch.full((heads, T), 7.0, device=DEV)
    o, lse = B.attention_packed(q, k, v, cu, heads, kv, impl=impl, out=out, lse=lse)
    grads = [torch.full((T, w * hs), 7.0, dtype=dtype, device=DEV) for w in (heads, kv, kv)]
    B.attention_packed_backward(q, k, v, o, lse, d_o, cu, heads, kv, impl=impl, dq=grads[0], dk=grads[1], dv=grads[2])
    assert B.device_status() == 0
    for t in [o] + grads:
        assert bool((t[:gap] == 7).all()) and bool((t[end:] == 7).all())
    assert bool((lse[:, :gap] == 7).all()) and bool((lse[:, end:] == 7).all())
    ro, rl, bo, bl = R.forward(*clean[:3], lens, heads, kv, gap)
    assert bool(((o.double() - ro).abs() <= bo)[gap:end].all())
    assert bool(((lse.double() - rl).abs() <= bl)[:, gap:end].all())
    want, bounds = R.backward(*clean, lens, heads, kv, gap)
    for x, r, b in zip(grads, want, bounds):
        assert bool(((x.double() - r).abs() <= b)[gap:end].all())


@pytest.mark.parametrize("impl", [0, 2])
@pytest.mark.parametrize("hs,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (48, torch.float32)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_masked_infinities(hs, dtype, impl, bad):
    """A NaN or infinity in one sequence, at a late position: the other sequences (in the same tiles) and the earlier
    positions come out as if it were not there, forward and backward across sequences."""
    lens, heads, kv = [40, 60, 200, 30], 4, 2
    q, k, v, d_o = make(lens, heads, kv, hs, dtype, seed=6)
    cu = cu_of(lens)
    clean_o, clean_lse = B.attention_packed(q, k, v, cu, heads, kv, impl=impl)
    ro, rl, bo, bl = R.forward(q, k, v, lens, heads, kv)
    want, bounds = R.backward(q, k, v, d_o, lens, heads, kv)
    at = 40 + 60 + 150           # a position of the third sequence
    k, v = k.clone(), v.clone()
    k[at, 3] = bad
    v[at, 5] = bad
    o, lse = B.attention_packed(q, k, v, cu, heads, kv, impl=impl)
    fine = [i for i in range(sum(lens)) if i < at or i >= 300]
    assert bool(((o.double() - ro).abs() <= bo)[fine].all())
    assert bool(((lse.double() - rl).abs() <= bl)[:, fine].all())
    # every later row of the third sequence sees it
    assert not bool(torch.isfinite(o[at:300, :hs].float()).all(1).any())
    dq, dk, dv = B.attention_packed_backward(q, k, v, o, lse, d_o, cu, heads, kv, impl=impl)
    others = [i for i in range(sum(lens)) if i < 100 or i >= 300]
    for x, r, b in zip((dq, dk, dv), want, bounds):
        assert bool(((x.double() - r).abs() <= b)[others].all())
    # query rows before the position do not see it either
    assert bool(((dq.double() - want[0]).abs() <= bounds[0])[100:at].all())
    assert B.device_status() == 0
    assert clean_o.shape == o.shape and clean_lse.shape == lse.shape


@pytest.mark.parametrize("impl", [0, 2])
@pytest.mark.parametrize("hs,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (48, torch.float32), (32, torch.bfloat16)])
def test_scores_of_minus_infinity(hs, dtype, impl):
    """Keys whose scores are minus infinity have no weight, however many of them a row meets first."""
    heads, kv, dead, n = 4, 2, 200, 320
    q, k, v, _ = make([n], heads, kv, hs, dtype, seed=9)
    q, k, v = q.abs() + 0.1, k.clone(), v.clone()
    k[:dead] = 0.0
    k.view(n, kv, hs)[:dead, :, 3] = -math.inf
    o, lse = B.attention_packed(q, k, v, cu_of([n]), heads, kv, impl=impl)
    rest = [t[dead:].contiguous() for t in (q, k, v)]
    ro, rl, bo, bl = R.forward(*rest, [n - dead], heads, kv)
    assert bool(((o[dead:].double() - ro).abs() <= bo).all())
    assert bool(((lse[:, dead:].double() - rl).abs() <= bl).all())
    assert bool(o[:dead].isnan().all()) and bool((lse[:, :dead] == -math.inf).all())
    assert B.device_status() == 0


def test_strides_and_alignment():
    """Views with odd pitches and offsets take the CUDA-core kernel and give the same values."""
    lens, heads, kv, hs = [50, 90], 2, 1, 64
    g = torch.Generator(device=DEV).manual_seed(1)
    base = torch.randn(140, 4 * 64 + 3, generator=g, device=DEV).bfloat16()
    q, k, v = base[:, 1:129], base[:, 129:193], base[:, 194:258]
    o, lse = check_fwd(q, k, v, lens, heads, kv)
    d_o = torch.randn(140, 128, generator=g, device=DEV).bfloat16()
    wide = torch.zeros(140, 200, device=DEV).bfloat16()
    dq, dk, dv = B.attention_packed_backward(q, k, v, o, lse, d_o, cu_of(lens), heads, kv, dq=wide[:, 3:131])
    want, bounds = R.backward(q, k, v, d_o, lens, heads, kv)
    for x, r, b in zip((dq, dk, dv), want, bounds):
        assert bool(((x.double() - r).abs() <= b).all())
    assert bool((wide[:, :3] == 0).all()) and bool((wide[:, 131:] == 0).all())


def test_equals_rectangular_attention():
    """Equal lengths and as many key heads as query heads: the rectangular entry point computes the same thing."""
    b, s, heads, hs = 3, 200, 4, 64
    q, k, v, d_o = make([s] * b, heads, heads, hs, torch.bfloat16, seed=8)
    o, lse = B.attention_packed(q, k, v, cu_of([s] * b), heads)
    o2, lse2 = B.attention(q, k, v, b, s, heads)
    # both are within the bound of the exact result (weights and outputs rounded to bf16), so within twice that of each
    # other; a fixed 2^-7 (1 + |o|) was no bound, as sum p|v| exceeds 1 where few keys are seen
    bound = R.forward(q, k, v, [s] * b, heads, heads)[2]
    assert bool(((o.double() - o2.double()).abs() <= 2 * bound).all())
    assert torch.allclose(lse.view(heads, b, s).transpose(0, 1), lse2, rtol=1e-5, atol=1e-5)


def test_gradient_against_differences():
    """fp32 gradients against central differences of the 64-bit forward along random directions."""
    lens, heads, kv, hs = [9, 1, 20], 4, 2, 16
    q, k, v, d_o = make(lens, heads, kv, hs, torch.float32, seed=2)
    cu = cu_of(lens)
    o, lse = B.attention_packed(q, k, v, cu, heads, kv)
    grads = B.attention_packed_backward(q, k, v, o, lse, d_o, cu, heads, kv)
    value = lambda a, b, c: float((R.forward(a, b, c, lens, heads, kv)[0] * d_o.double()).sum())
    g = torch.Generator(device=DEV).manual_seed(11)
    # central differences are off by O(h^2) and by the forward's 2^-53 / h; the gradient by its bound times |direction|
    want, bounds = R.backward(q, k, v, d_o, lens, heads, kv)
    h = 1e-5
    for i, (x, grad) in enumerate(zip((q, k, v), grads)):
        d = torch.randn(x.shape, generator=g, device=DEV, dtype=torch.float64)
        args = [t.double() for t in (q, k, v)]
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + h * d, args[i] - h * d
        R.U[torch.float64] = 0.0
        try:
            diff = (value(*up) - value(*down)) / (2 * h)
        finally:
            del R.U[torch.float64]
        got = float((grad.double() * d).sum())
        assert abs(got - diff) <= float((bounds[i] * d.abs()).sum()) + 1e-6 * (1 + abs(diff))


@pytest.mark.parametrize("lens,heads,kv_heads,hs", [
    ([300, 0, 1100, 7], 8, 4, 64), ([300, 0, 1100, 7], 8, 2, 128),         # two CTAs share a key tile
    ([700, 300], 6, 1, 128), ([129], 4, 2, 64), ([1, 1, 2], 2, 1, 128),
    ([400, 100] * 20, 16, 8, 64), ([30] * 100, 32, 16, 64), ([600], 9, 3, 128)])  # they do not
def test_backward_of_grouped_heads(lens, heads, kv_heads, hs):
    q, k, v, d_o = make(lens, heads, kv_heads, hs, torch.bfloat16, seed=21, gap=3, tail=5)
    cu = cu_of(lens, 3)
    o, lse = B.attention_packed(q, k, v, cu, heads, kv_heads)
    marks = [torch.full(x.shape, 7.0, dtype=x.dtype, device=DEV) for x in (q, k, v)]
    got = B.attention_packed_backward(q, k, v, o, lse, d_o, cu, heads, kv_heads, dq=marks[0], dk=marks[1], dv=marks[2])
    assert B.device_status() == 0
    want, bounds = R.backward(q, k, v, d_o, lens, heads, kv_heads, 3)
    for name, x, r, b in zip(("dq", "dk", "dv"), got, want, bounds):
        err = (x.double() - r).abs()[3:-5]
        assert bool((err <= b[3:-5]).all()), (name, float((err / b[3:-5]).max()))
        assert bool((x[:3] == 7).all() and (x[-5:] == 7).all())
    again = B.attention_packed_backward(q, k, v, o, lse, d_o, cu, heads, kv_heads)
    assert all(torch.equal(x[3:-5], y[3:-5]) for x, y in zip(got, again))


@pytest.mark.parametrize("impl", [0, 2])
@pytest.mark.parametrize("lens", [[1] * 300, [1, 130, 1, 1, 63, 1, 200, 2, 1, 1]])
@pytest.mark.parametrize("hs,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (48, torch.float32), (32, torch.bfloat16)])
def test_a_row_that_sees_itself_alone(hs, dtype, lens, impl):
    # its softmax is the constant 1: no gradient of its scores, not even a rounding error's
    heads, kv_heads = 6, 2
    q, k, v, d_o = make(lens, heads, kv_heads, hs, dtype, seed=12)
    cu = cu_of(lens)
    o, lse = B.attention_packed(q, k, v, cu, heads, kv_heads, impl=impl)
    dq, dk, dv = B.attention_packed_backward(q, k, v, o, lse, d_o, cu, heads, kv_heads, impl=impl)
    assert B.device_status() == 0
    starts = cu[:-1].long()
    assert not bool(dq[starts].any())
    single = starts[torch.tensor(lens, device=DEV) == 1]
    assert not bool(dk[single].any())
    assert bool(dq.isfinite().all() and dk.isfinite().all() and dv.isfinite().all())


@pytest.mark.parametrize("hs,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (48, torch.float32)])
def test_repeats_to_the_bit(hs, dtype):
    lens, heads, kv = [300, 7, 129], 6, 2
    q, k, v, d_o = make(lens, heads, kv, hs, dtype, seed=5)
    cu = cu_of(lens)
    o, lse = B.attention_packed(q, k, v, cu, heads, kv)
    first = (o, lse) + B.attention_packed_backward(q, k, v, o, lse, d_o, cu, heads, kv)
    for _ in range(3):
        o, lse = B.attention_packed(q, k, v, cu, heads, kv)
        again = (o, lse) + B.attention_packed_backward(q, k, v, o, lse, d_o, cu, heads, kv)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("hs", [64, 128])
def test_captured_and_replayed_on_another_stream(hs):
    """A training pass (forward, backward) captured into a graph and replayed on new inputs, while an eager call runs
    beside it on its own stream."""
    lens, heads, kv = [200, 90], 4, 2
    q, k, v, d_o = (t.clone() for t in make(lens, heads, kv, hs, torch.bfloat16, seed=5))
    cu = cu_of(lens)
    o, lse = B.attention_packed(q, k, v, cu, heads, kv)
    B.attention_packed_backward(q, k, v, o, lse, d_o, cu, heads, kv)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go, glse = B.attention_packed(q, k, v, cu, heads, kv)
        grads = B.attention_packed_backward(q, k, v, go, glse, d_o, cu, heads, kv)
    q2, k2, v2, d2 = make(lens, heads, kv, hs, torch.bfloat16, seed=77)
    for a, b in zip((q, k, v, d_o), (q2, k2, v2, d2)):
        a.copy_(b)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        eo, elses = B.attention_packed(q2, k2, v2, cu, heads, kv)
        eager = B.attention_packed_backward(q2, k2, v2, eo, elses, d2, cu, heads, kv)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip((go, glse) + grads, (eo, elses) + eager):
        assert torch.equal(a, b)
    assert B.device_status() == 0


def test_empty_calls():
    q, k, v, d_o = make([], 2, 1, 64, torch.bfloat16)
    cu = torch.zeros(1, dtype=torch.int32, device=DEV)
    o, lse = B.attention_packed(q, k, v, cu, 2, 1)
    assert o.shape == (0, 128) and lse.shape == (2, 0)
    dq, dk, dv = B.attention_packed_backward(q, k, v, o, lse, d_o, cu, 2, 1)
    assert dq.shape == (0, 128) and dk.shape == (0, 64)
    # rows but only empty sequences: nothing is written
    q, k, v, _ = make([4], 2, 1, 64, torch.bfloat16)
    out = torch.full((4, 128), 3.0, device=DEV).bfloat16()
    B.attention_packed(q, k, v, torch.zeros(5, dtype=torch.int32, device=DEV), 2, 1, out=out)
    assert bool((out == 3).all())


def test_refusals():
    q, k, v, d_o = make([8], 4, 2, 64, torch.bfloat16)
    cu = cu_of([8])
    for call, status in [
        (lambda: B.attention_packed(q, k, v, cu, 3, 2), 2),
        (lambda: B.attention_packed(q, k, v, cu, 4, 3), 2),
        (lambda: B.attention_packed(q, k, v[:7], cu, 4, 2), 2),
        (lambda: B.attention_packed(q, k.float(), v, cu, 4, 2), 3),
        (lambda: B.attention_packed(q.half(), k.half(), v.half(), cu, 4, 2), 3),
        (lambda: B.attention_packed(q, k, v, cu.long(), 4, 2), 3),
        (lambda: B.attention_packed(q, k, v, cu.cpu(), 4, 2), 1),
        (lambda: B.attention_packed(q, k, v, cu, 4, 2, impl=3), 1),
        (lambda: B.attention_packed(q[:, :160].contiguous(), k[:, :80].contiguous(), v[:, :80].contiguous(), cu, 4, 2), 2),
        (lambda: B.attention_packed(q.float(), k.float(), v.float(), cu, 4, 2, impl=1), 10),
        (lambda: B.attention_packed(q[:1].expand(8, 256), k, v, cu, 4, 2), 2),
        (lambda: B.attention_packed(q, k, v, cu, 4, 2, lse=torch.zeros(8, 4, device=DEV)), 2),
    ]:
        with pytest.raises(B.B200Error) as e:
            call()
        assert e.value.status == status
