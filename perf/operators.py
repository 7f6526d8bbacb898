"""Measured cases of the packed-prompt attention, the 4-bit key/value cache and the page copies.

Each case is one call (or the pair append + read back) a user makes of ``b200_llama``.  With ``own`` false the same
result is computed from elementary torch operations in 32 bits; with ``own`` true the framework's kernels run.

Layouts: q, o ``[T, n_heads * hs]``; k, v ``[T, n_kv_heads * hs]``; the sequences of a packed batch lie one behind the
other and ``cu_seqlens`` int32 ``[n_seqs + 1]`` names their first rows.  A 4-bit cache layer is ``codes`` uint8
``[2, n_pages, n_kv_heads, page_size, hs // 2]`` (keys, values; element 2i in the low half of byte i) with ``params``
bf16 ``[2, n_pages, n_kv_heads, page_size, 2]`` (scale, minimum): a row stands for ``minimum + scale * code``.
"""
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _lib():
    path = os.path.join(_ROOT, "enzyme-jax_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import b200_llama
    return b200_llama


# ---- cases -----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a handful of very short fp32 prompts at the 15M-parameter shape (6 heads of 48): latency counts
        dict(name="prompt_tiny_fp32", op="fwd", dtype="float32", heads=6, kv_heads=6, hs=48, n_seqs=3, max_len=17, lens="ragged"),
        # a serving batch of prompts of mixed lengths at the 7B width, four query heads to a key head
        dict(name="prompt_ragged_7b", op="fwd", dtype="bfloat16", heads=32, kv_heads=8, hs=128, n_seqs=24, max_len=2048, lens="ragged"),
        # two long prompts at the 7B width
        dict(name="prompt_long_7b", op="fwd", dtype="bfloat16", heads=32, kv_heads=8, hs=128, n_seqs=2, max_len=8192, lens="even"),
        # training on packed documents at the 110M shape (12 heads of 64), a micro-batch of 8 x 1024 tokens
        dict(name="train_110m", op="bwd", dtype="bfloat16", heads=12, kv_heads=12, hs=64, n_seqs=8, max_len=1024, lens="even"),
        # training on packed documents of mixed lengths at the 7B width with grouped heads
        dict(name="train_ragged_7b", op="bwd", dtype="bfloat16", heads=32, kv_heads=8, hs=128, n_seqs=12, max_len=2048, lens="ragged"),
        # the cache write of one decode step: one new row for each of 64 sequences
        dict(name="append_step_7b", op="append", dtype="bfloat16", kv_heads=32, hs=128, n_seqs=64, max_len=1, lens="even", before=4095, page=64),
        # the cache write of a batch of prompts, mixed lengths
        dict(name="append_prompts_7b", op="append", dtype="bfloat16", kv_heads=8, hs=128, n_seqs=24, max_len=2048, lens="ragged", before=0, page=64),
        # one user's chat: a single sequence of a few hundred tokens
        dict(name="decode_one", op="decode", dtype="bfloat16", heads=32, kv_heads=8, hs=128, n_seqs=1, max_len=500, lens="even", page=64),
        # the 7B decode configuration: 64 sequences of 4096 cached tokens, every head with its own keys
        dict(name="decode_7b", op="decode", dtype="bfloat16", heads=32, kv_heads=32, hs=128, n_seqs=64, max_len=4096, lens="even", page=64),
        # sequences of very different lengths in one step, grouped heads
        dict(name="decode_ragged", op="decode", dtype="bfloat16", heads=32, kv_heads=8, hs=128, n_seqs=16, max_len=32768, lens="ragged", page=64),
        # beams or samples that part: the partly filled last pages of 16 sequences are copied, all layers of the 7B shape
        dict(name="fork_last_pages_7b", op="pages", mode="fork", layers=32, kv_heads=32, hs=128, page=64, n_pages=48, n=16),
        # a small pool is compacted: live pages move to the front and the page table follows (110M shape)
        dict(name="compact_110m", op="pages", mode="compact", layers=12, kv_heads=12, hs=64, page=64, n_pages=64, n=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["fwd", "fwd", "bwd", "bwd", "append", "decode", "decode", "pages"])
    if op in ("fwd", "bwd"):
        kind = rng.choice(["tensor", "tensor", "tensor", "small"])
        if kind == "tensor":  # the training and serving shapes
            dtype, hs = "bfloat16", rng.choice([64, 128])
            kv_heads = rng.choice([1, 2, 4, 8])
            heads = kv_heads * rng.choice([1, 2, 3, 4])
            max_len = _log(rng, 1, 4096)
            n_seqs = max(1, min(_log(rng, 1, 128), 8192 // max_len))
        else:                 # the exact and the small-head shapes
            dtype, hs = rng.choice(["float32", "float32", "bfloat16"]), rng.choice([16, 32, 48, 64, 128])
            kv_heads = rng.choice([1, 2, 6])
            heads = kv_heads * rng.choice([1, 2, 3])
            max_len = _log(rng, 1, 512)
            n_seqs = max(1, min(_log(rng, 1, 32), 2048 // max_len))
        return dict(op=op, dtype=dtype, heads=heads, kv_heads=kv_heads, hs=hs, n_seqs=n_seqs, max_len=max_len,
                    lens=rng.choice(["ragged", "even"]))
    if op == "append":
        hs = rng.choice([32, 48, 64, 128])
        max_len = _log(rng, 1, 2048)
        return dict(op=op, dtype="bfloat16", kv_heads=rng.choice([1, 2, 6, 8, 32]), hs=hs,
                    n_seqs=max(1, min(_log(rng, 1, 128), 8192 // max_len)), max_len=max_len,
                    lens=rng.choice(["ragged", "even"]), before=rng.choice([0, rng.randrange(0, 3000)]),
                    page=rng.choice([16, 32, 64, 128]))
    if op == "decode":
        kind = rng.choice(["tensor", "tensor", "tensor", "small"])
        if kind == "tensor":
            dtype, hs, page = "bfloat16", rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
            kv_heads = rng.choice([1, 2, 4, 8, 32])
            heads = kv_heads * (1 if kv_heads == 32 else rng.choice([1, 2, 4, 6, 8]))
            max_len = _log(rng, 1, 32768)
            n_seqs = max(1, min(_log(rng, 1, 128), 4194304 // (max_len * kv_heads)))
        else:
            dtype, hs, page = rng.choice(["float32", "bfloat16"]), rng.choice([32, 48, 64, 128]), rng.choice([12, 16, 64])
            kv_heads = rng.choice([1, 2, 6])
            heads = kv_heads * rng.choice([1, 2, 3])
            max_len = _log(rng, 1, 2048)
            n_seqs = _log(rng, 1, 16)
        return dict(op=op, dtype=dtype, heads=heads, kv_heads=kv_heads, hs=hs, n_seqs=n_seqs, max_len=max_len,
                    lens=rng.choice(["ragged", "even"]), page=page)
    hs = rng.choice([48, 64, 128])
    n_pages = rng.randrange(8, 65)
    return dict(op=op, mode=rng.choice(["fork", "compact"]), layers=rng.choice([1, 6, 12]), kv_heads=rng.choice([2, 6, 8, 12]),
                hs=hs, page=rng.choice([12, 16, 64, 128]), n_pages=n_pages, n=rng.randrange(1, n_pages // 3 + 1))


# ---- sizes -----------------------------------------------------------------------------------------------------------
def _lengths(case):
    """Sequence lengths of a case: all equal, or spread over 1 .. max_len (on a log scale) with the longest one present."""
    n, m = case["n_seqs"], case["max_len"]
    if case["lens"] == "even":
        return [m] * n
    rng = random.Random(n * 1000003 + m)
    out = [m] + [max(1, min(m, int(math.exp(rng.uniform(math.log(max(1, m / 64)), math.log(m + 0.5)))))) for _ in range(n - 1)]
    rng.shuffle(out)
    return out


def _esize(case):
    return 4 if case["dtype"] == "float32" else 2


def _page_rows(case):
    """Filled rows of the pages a fork copies (the last page of a sequence is partly filled)."""
    rng = random.Random(case["n"] * 7919 + case["page"])
    return [rng.randrange(1, case["page"] + 1) for _ in range(case["n"])]


def work(case):
    op = case["op"]
    if op in ("fwd", "bwd"):
        lens = _lengths(case)
        t, e, h, hk, hs = sum(lens), _esize(case), case["heads"], case["kv_heads"], case["hs"]
        pairs = sum(n * (n + 1) // 2 for n in lens)
        stats = 4 * h * t + 4 * (len(lens) + 1)
        if op == "fwd":   # q, k, v in; o, lse out; two products
            return {"bytes": t * hs * e * (2 * h + 2 * hk) + stats, "flops": 4 * pairs * h * hs}
        # q, k, v, o, d_o, lse in; dq, dk, dv out; five products
        return {"bytes": t * hs * e * (4 * h + 4 * hk) + stats, "flops": 10 * pairs * h * hs}
    if op == "append":
        t, hk, hs, e = sum(_lengths(case)), case["kv_heads"], case["hs"], _esize(case)
        held = t * hk * (hs + 8)   # codes and (scale, minimum) of a key and a value row
        return {"bytes": 2 * t * hk * hs * e + 2 * held + 2 * t * hk * hs * e, "flops": 2 * t * hk * hs * 6}
    if op == "decode":
        lens = _lengths(case)
        t, h, hk, hs, e = sum(lens), case["heads"], case["kv_heads"], case["hs"], _esize(case)
        return {"bytes": t * hk * (hs + 8) + 2 * len(lens) * h * hs * e, "flops": 4 * t * h * hs}
    rows = sum(_page_rows(case)) if case["mode"] == "fork" else case["n"] * case["page"]
    return {"bytes": 2 * 2 * case["layers"] * rows * case["kv_heads"] * case["hs"] * 2, "flops": 0}


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _cu(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def _bf16_down(x):
    """Rounds fp32 to the next bf16 value at or below it."""
    b = x.view(torch.int32)
    cut = b & -65536
    return torch.where((b < 0) & (cut != b), cut + 65536, cut).view(torch.float32)


def _bf16_up(x):
    """Rounds a non-negative fp32 to the next bf16 value at or above it."""
    b = x.view(torch.int32)
    cut = b & -65536
    return torch.where(cut != b, cut + 65536, cut).view(torch.float32)


def _quantise(rows):
    """fp32 [..., hs] -> (codes as fp32 0..15, scale, minimum): 16 evenly spaced values from the row's minimum (rounded
    down to bf16) that reach its maximum (scale rounded up to bf16)."""
    lo = _bf16_down(rows.amin(-1, keepdim=True))
    # divided by a tensor: a division by a plain number becomes a product with its rounded reciprocal
    scale = _bf16_up((rows.amax(-1, keepdim=True) - lo) / torch.full_like(lo, 15.0))
    safe = torch.where(scale > 0, scale, torch.ones_like(scale))
    codes = torch.round((rows - lo) / safe).clamp_(0.0, 15.0)
    return codes, scale, lo


def _pack(codes):
    c = codes.to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def _tables(case, lens, g):
    """Shuffled page table [n_seqs, max_pages] and the number of pages of the pool."""
    page = case["page"]
    need = [max(1, -(-n // page)) for n in lens]
    width = max(need)
    total = sum(need) + 2
    perm = torch.randperm(total, generator=g, device="cuda")
    idx, live, at = [], [], 0
    for n in need:
        idx.append([at + min(i, n - 1) for i in range(width)])
        at += n
    return perm[torch.tensor(idx, device="cuda")].int(), total


def _plain_forward(q, k, v, lens, heads, kv_heads, hs, row_block=2048):
    """fp32 outputs [T, heads, hs] and log-sum-exps [heads, T]."""
    t = q.shape[0]
    group = heads // kv_heads
    o = torch.empty(t, heads, hs, device=q.device)
    lse = torch.empty(heads, t, device=q.device)
    at = 0
    for n in lens:
        ks = k[at:at + n].view(n, kv_heads, hs).float().permute(1, 2, 0)
        vs = v[at:at + n].view(n, kv_heads, hs).float().permute(1, 0, 2)
        for r0 in range(0, n, row_block):
            r1 = min(n, r0 + row_block)
            qs = q[at + r0:at + r1].view(r1 - r0, kv_heads, group, hs).float().permute(1, 2, 0, 3)
            s = torch.matmul(qs, ks[:, None, :, :r1]) * (hs ** -0.5)
            hidden = torch.arange(r1, device=q.device)[None, :] > torch.arange(r0, r1, device=q.device)[:, None]
            s = s.masked_fill(hidden, float("-inf"))
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - top)
            total = p.sum(-1, keepdim=True)
            out = torch.matmul(p, vs[:, None, :r1]) / total
            o[at + r0:at + r1] = out.permute(2, 0, 1, 3).reshape(r1 - r0, heads, hs)
            lse[:, at + r0:at + r1] = (top + torch.log(total)).squeeze(-1).reshape(heads, r1 - r0)
        at += n
    return o, lse


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "pages":
        layers, hk, page, hs, n_pages, n = (case[k] for k in ("layers", "kv_heads", "page", "hs", "n_pages", "n"))
        pool = _randn(g, layers, 2, n_pages, hk, page, hs, dtype=torch.bfloat16)
        state = dict(case=case, pool=pool)
        if case["mode"] == "fork":
            perm = torch.randperm(n_pages, generator=g, device="cuda").int()
            state["src"], state["dst"] = perm[:n].contiguous(), perm[n:2 * n].contiguous()
            state["rows_host"] = _page_rows(case)
            state["rows"] = torch.tensor(state["rows_host"], dtype=torch.int32, device="cuda")
        else:
            # live pages: all but the n free ones in the front part; the last n pages are live and move into them
            front = torch.randperm(n_pages - n, generator=g, device="cuda")[:n]
            state["dst"] = front.sort().values.int()
            state["src"] = torch.arange(n_pages - n, n_pages, device="cuda", dtype=torch.int32)
            page_map = torch.arange(n_pages, device="cuda", dtype=torch.int32)
            page_map[state["src"].long()] = state["dst"]
            state["page_map"] = page_map
            live = torch.ones(n_pages, dtype=torch.bool, device="cuda")
            live[state["dst"].long()] = False
            ids = torch.nonzero(live)[:, 0].int()
            state["table"] = ids[torch.randperm(ids.numel(), generator=g, device="cuda")].view(1, -1).contiguous()
        return state
    dtype = getattr(torch, case["dtype"])
    lens = _lengths(case)
    hk, hs = case["kv_heads"], case["hs"]
    state = dict(case=case, lens=lens)
    if op in ("fwd", "bwd"):
        h, t = case["heads"], sum(lens)
        qkv = _randn(g, t, (h + 2 * hk) * hs, dtype=dtype)   # the projection's output: q, k and v side by side
        state["q"], state["k"], state["v"] = qkv[:, :h * hs], qkv[:, h * hs:(h + hk) * hs], qkv[:, (h + hk) * hs:]
        state["cu"] = _cu(lens)
        if op == "bwd":
            o, lse = _plain_forward(state["q"], state["k"], state["v"], lens, h, hk, hs)
            state["o"], state["lse"] = o.view(t, h * hs).to(dtype), lse
            state["d_o"] = _randn(g, t, h * hs, dtype=dtype)
        return state
    if op == "append":
        t = sum(lens)
        kv = _randn(g, t, 2 * hk * hs, dtype=dtype)
        state["k"], state["v"] = kv[:, :hk * hs], kv[:, hk * hs:]
        state["cu"] = _cu(lens)
        state["before"] = torch.full((len(lens),), case["before"], dtype=torch.int32, device="cuda")
        state["table"], n_pages = _tables(case, [n + case["before"] for n in lens], g)
        state["codes"] = torch.zeros(2, n_pages, hk, case["page"], hs // 2, dtype=torch.uint8, device="cuda")
        state["params"] = torch.zeros(2, n_pages, hk, case["page"], 2, dtype=torch.bfloat16, device="cuda")
        return state
    state["table"], n_pages = _tables(case, lens, g)
    page = case["page"]
    codes = torch.empty(2, n_pages, hk, page, hs // 2, dtype=torch.uint8, device="cuda")
    params = torch.empty(2, n_pages, hk, page, 2, dtype=torch.bfloat16, device="cuda")
    step = max(1, (1 << 26) // (hk * page * hs))
    for i in range(2):
        for p in range(0, n_pages, step):
            c, s, lo = _quantise(_randn(g, min(step, n_pages - p), hk, page, hs))
            codes[i, p:p + step] = _pack(c)
            params[i, p:p + step] = torch.cat((s, lo), -1).to(torch.bfloat16)
    state["codes"], state["params"] = codes, params
    state["ctx"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    state["q"] = _randn(g, len(lens), case["heads"] * hs, dtype=dtype)
    return state


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        b = _lib()
        if op == "fwd":
            o, lse = b.attention_packed(state["q"], state["k"], state["v"], state["cu"], case["heads"], case["kv_heads"])
            return {"o": o, "lse": lse}
        if op == "bwd":
            dq, dk, dv = b.attention_packed_backward(state["q"], state["k"], state["v"], state["o"], state["lse"],
                                                     state["d_o"], state["cu"], case["heads"], case["kv_heads"])
            return {"dq": dq, "dk": dk, "dv": dv}
        if op == "append":
            b.kv4_append(state["k"], state["v"], state["codes"], state["params"], state["table"], state["cu"], state["before"])
            k, v = b.kv4_read(state["codes"], state["params"], state["table"], state["cu"], state["before"], state["k"].shape[0],
                              dtype=state["k"].dtype)
            return {"k": k, "v": v}
        if op == "decode":
            return {"o": b.attention_decode_kv4(state["q"], state["codes"], state["params"], state["table"], state["ctx"],
                                                case["heads"])}
        if case["mode"] == "fork":
            b.copy_pages(state["pool"], state["src"], state["dst"], rows=state["rows"])
            return {"pool": state["pool"]}
        b.compact_pages(state["pool"], state["src"], state["dst"], state["table"], state["page_map"])
        return {"pool": state["pool"], "table": state["table"]}
    if op == "fwd":
        h, hs = case["heads"], case["hs"]
        o, lse = _plain_forward(state["q"], state["k"], state["v"], state["lens"], h, case["kv_heads"], hs)
        return {"o": o.view(-1, h * hs).to(state["q"].dtype), "lse": lse}
    if op == "bwd":
        return _plain_backward(state)
    if op == "append":
        return _plain_append(state)
    if op == "decode":
        return _plain_decode(state)
    src, dst = state["src"].long(), state["dst"].long()
    if case["mode"] == "fork":
        keep = torch.arange(case["page"], device="cuda")[None, :] < state["rows"][:, None]
        keep = keep[None, None, :, None, :, None]
        state["pool"][:, :, dst] = torch.where(keep, state["pool"][:, :, src], state["pool"][:, :, dst])
        return {"pool": state["pool"]}
    state["pool"][:, :, dst] = state["pool"][:, :, src]
    state["table"].copy_(state["page_map"][state["table"].long()])
    return {"pool": state["pool"], "table": state["table"]}


def _plain_backward(state, row_block=2048):
    case = state["case"]
    h, hk, hs = case["heads"], case["kv_heads"], case["hs"]
    group, scale = h // hk, hs ** -0.5
    q, k, v, d_o = state["q"], state["k"], state["v"], state["d_o"]
    t, dev = q.shape[0], q.device
    dq = torch.empty(t, h, hs, device=dev)
    dk = torch.zeros(t, hk, hs, device=dev)
    dv = torch.zeros(t, hk, hs, device=dev)
    at = 0
    for n in state["lens"]:
        ks = k[at:at + n].view(n, hk, hs).float().permute(1, 0, 2)
        vs = v[at:at + n].view(n, hk, hs).float().permute(1, 0, 2)
        for r0 in range(0, n, row_block):
            r1 = min(n, r0 + row_block)
            kk, vv = ks[:, None, :r1], vs[:, None, :r1]
            qs = q[at + r0:at + r1].view(r1 - r0, hk, group, hs).float().permute(1, 2, 0, 3)
            gs = d_o[at + r0:at + r1].view(r1 - r0, hk, group, hs).float().permute(1, 2, 0, 3)
            ls = state["lse"][:, at + r0:at + r1].reshape(hk, group, r1 - r0, 1)
            s = torch.matmul(qs, kk.transpose(-1, -2)) * scale
            hidden = torch.arange(r1, device=dev)[None, :] > torch.arange(r0, r1, device=dev)[:, None]
            p = torch.exp(s - ls).masked_fill(hidden, 0.0)
            dp = torch.matmul(gs, vv.transpose(-1, -2))
            ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
            dq[at + r0:at + r1] = torch.matmul(ds, kk).permute(2, 0, 1, 3).reshape(r1 - r0, h, hs)
            dk[at:at + r1] += torch.matmul(ds.transpose(-1, -2), qs).sum(1).permute(1, 0, 2)
            dv[at:at + r1] += torch.matmul(p.transpose(-1, -2), gs).sum(1).permute(1, 0, 2)
        at += n
    return {"dq": dq.view(t, -1).to(q.dtype), "dk": dk.view(t, -1).to(k.dtype), "dv": dv.view(t, -1).to(v.dtype)}


def _places(state):
    """Page and row inside the page of every appended row."""
    page = state["case"]["page"]
    seq = torch.repeat_interleave(torch.arange(len(state["lens"]), device="cuda"),
                                  (state["cu"][1:] - state["cu"][:-1]).long(), output_size=state["k"].shape[0])
    pos = torch.arange(state["k"].shape[0], device="cuda") - state["cu"].long()[seq] + state["before"].long()[seq]
    return state["table"].long()[seq, pos // page], pos % page


def _plain_append(state):
    case = state["case"]
    hk, hs = case["kv_heads"], case["hs"]
    pages, rows = _places(state)
    out = {}
    for i, name in enumerate(("k", "v")):
        x = state[name].view(-1, hk, hs).float()
        c, s, lo = _quantise(x)
        state["codes"][i, pages, :, rows] = _pack(c)
        state["params"][i, pages, :, rows] = torch.cat((s, lo), -1).to(torch.bfloat16)
        held, prm = state["codes"][i, pages, :, rows], state["params"][i, pages, :, rows].float()
        back = torch.stack((held & 15, held >> 4), -1).view(-1, hk, hs).float() * prm[..., :1] + prm[..., 1:]
        out[name] = back.view(-1, hk * hs).to(state[name].dtype)
    return out


def _plain_decode(state):
    case = state["case"]
    h, hk, hs, page = case["heads"], case["kv_heads"], case["hs"], case["page"]
    q = state["q"].view(-1, hk, h // hk, hs).float()
    out = torch.empty(len(state["lens"]), hk, h // hk, hs, device="cuda")
    for b, n in enumerate(state["lens"]):
        pages = state["table"][b, :-(-n // page)].long()
        rows = []
        for i in range(2):
            c = state["codes"][i, pages].transpose(0, 1).reshape(hk, -1, hs // 2)[:, :n]
            prm = state["params"][i, pages].transpose(0, 1).reshape(hk, -1, 2)[:, :n].float()
            rows.append(torch.stack((c & 15, c >> 4), -1).view(hk, n, hs).float() * prm[..., :1] + prm[..., 1:])
        s = torch.matmul(q[b], rows[0].transpose(-1, -2)) * (hs ** -0.5)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        out[b] = torch.matmul(p, rows[1]) / p.sum(-1, keepdim=True)
    return {"o": out.view(len(state["lens"]), h * hs).to(state["q"].dtype)}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------
def exact(case, seed):
    op = case["op"]
    if op == "append":
        return _exact_append(prepare(case, seed))
    if op == "pages":
        return _exact_pages(prepare(case, seed))
    state = prepare(case, seed)
    if op == "decode":
        return _exact_decode(state)
    # one (sequence, query head) at a time, gradients by the chain rule on the normalised probabilities
    h, hk, hs, group = case["heads"], case["kv_heads"], case["hs"], case["heads"] // case["kv_heads"]
    t = state["q"].shape[0]
    f64 = dict(dtype=torch.float64, device="cuda")
    if op == "fwd":
        o, lse = torch.empty(t, h * hs, **f64), torch.empty(h, t, **f64)
    else:
        dq, dk, dv = torch.zeros(t, h * hs, **f64), torch.zeros(t, hk * hs, **f64), torch.zeros(t, hk * hs, **f64)
    first = 0
    for n in state["lens"]:
        span = slice(first, first + n)
        after = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
        for i in range(h):
            qc, kc = slice(i * hs, (i + 1) * hs), slice((i // group) * hs, (i // group + 1) * hs)
            qi, ki, vi = state["q"][span, qc].double(), state["k"][span, kc].double(), state["v"][span, kc].double()
            logits = (qi @ ki.T) / math.sqrt(hs)
            logits[after] = -math.inf
            norm = torch.logsumexp(logits, 1)
            prob = (logits - norm[:, None]).exp_()
            if op == "fwd":
                o[span, qc] = prob @ vi
                lse[i, span] = norm
            else:
                go = state["d_o"][span, qc].double()
                dv[span, kc] += prob.T @ go
                gp = go @ vi.T
                gl = prob * (gp - ((prob @ vi) * go).sum(1, keepdim=True)) / math.sqrt(hs)
                dq[span, qc] = gl @ ki
                dk[span, kc] += gl.T @ qi
        first += n
    return {"o": o, "lse": lse} if op == "fwd" else {"dq": dq, "dk": dk, "dv": dv}


def _exact_append(state):
    case = state["case"]
    out = {}
    for name in ("k", "v"):
        x = state[name].double().view(-1, case["kv_heads"], case["hs"])
        low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
        # inputs of 16 bits: the minimum is such a number itself; the scale goes up to the next one of 8 significant bits
        frac, expo = torch.frexp((high - low) / torch.full_like(low, 15.0))
        scale = torch.ldexp(torch.ceil(frac * 256.0) / 256.0, expo)
        code = torch.where(scale > 0, torch.round((x - low) / torch.where(scale > 0, scale, 1.0)), 0.0).clamp(0, 15)
        out[name] = (low + scale * code).view(-1, case["kv_heads"] * case["hs"])
    return out


def _exact_decode(state):
    case = state["case"]
    h, hk, hs, page = case["heads"], case["kv_heads"], case["hs"], case["page"]
    out = torch.empty(len(state["lens"]), h, hs, dtype=torch.float64, device="cuda")
    for b, n in enumerate(state["lens"]):
        at = torch.arange(n, device="cuda")
        pg, rw = state["table"][b].long()[at // page], at % page
        for j in range(hk):
            vals = []
            for i in range(2):
                byte = state["codes"][i, pg, j, rw].int()
                prm = state["params"][i, pg, j, rw].double()
                both = torch.empty(n, hs, dtype=torch.float64, device="cuda")
                both[:, 0::2], both[:, 1::2] = (byte % 16).double(), (byte // 16).double()
                vals.append(prm[:, 1:] + prm[:, :1] * both)
            heads = slice(j * (h // hk), (j + 1) * (h // hk))
            qs = state["q"][b].view(h, hs)[heads].double()
            out[b, heads] = torch.softmax(qs @ vals[0].T / math.sqrt(hs), -1) @ vals[1]
    return {"o": out.view(-1, h * hs)}


def _exact_pages(state):
    case, pool = state["case"], state["pool"]
    src, dst = state["src"].tolist(), state["dst"].tolist()
    want = pool.clone()
    for i, (a, b) in enumerate(zip(src, dst)):
        rows = state["rows_host"][i] if case["mode"] == "fork" else case["page"]
        want[:, :, b, :, :rows] = pool[:, :, a, :, :rows]
    if case["mode"] == "fork":
        return {"pool": want}
    moved = dict(zip(src, dst))
    table = [[moved.get(p, p) for p in row] for row in state["table"].tolist()]
    return {"pool": want, "table": torch.tensor(table, dtype=torch.int32, device="cuda")}
