"""The operators of a step that verifies a tree of drafted tokens over a paged cache, as timed cases.

Four operators, in the order in which such a step calls them behind the projection of its rows:

* `norm`: RMS norm of every q and k head and rotary positions in the same pass, with one axis of
  positions or several (time, height, width);
* `write`: K and V rows quantised as they are written into a paged cache, e4m3 values with a
  power of two for every head row;
* `tree`: attention of drafted tokens over the paged cache, in fp16 or e4m3: every row sees the
  context in front of the drafted tokens and its own ancestors among them;
* `read`: rows of the e4m3 cache read back (a prefix that another sequence goes on from).

Head counts, widths and lengths are those of the repository's own geometries: 14 query and 2 KV
heads of 64, 12 and 2 of 128, 32 and 8 of 128; blocks of 16 rows and more.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
E4M3 = torch.float8_e4m3fn
LOWEST, HIGHEST = -64, 32  # exponents of a head row of the e4m3 cache


def _tree(name, seqs, lo, hi, least, most, hq, hkv, d, pool, dtype, block=16, ragged=1):
    return dict(name=name, kind="tree", seqs=seqs, lo=lo, hi=hi, least=least, most=most, hq=hq,
                hkv=hkv, d=d, pool=pool, dtype=dtype, block=block, ragged=ragged)


def _rows(name, kind, tokens, hkv, d, dtype, block=16, fused=0):
    return dict(name=name, kind=kind, tokens=tokens, hkv=hkv, d=d, dtype=dtype, block=block,
                fused=fused)


def _norm(name, tokens, hq, hkv, d, rotary, axes, dtype, interleaved, far, gains=True):
    return dict(name=name, kind="norm", tokens=tokens, hq=hq, hkv=hkv, d=d, rotary=rotary,
                axes=axes, dtype=dtype, interleaved=interleaved, far=far, gains=gains)


def listed():
    return [
        # One conversation, a short prompt, a handful of drafted tokens: the smallest call.
        _tree("tree 1 user 7 drafts", 1, 300, 300, 7, 7, 12, 2, 128, "fp16", "fp16"),
        # A batch of conversations on a small model, from no draft at all (one row) to a dozen.
        _tree("tree 16 users heads of 64", 16, 100, 4096, 1, 12, 14, 2, 64, "fp16", "fp16"),
        # One user with a long document in front.
        _tree("tree context of 131072", 1, 131072, 131072, 24, 24, 32, 8, 128, "fp16", "fp16", 64),
        # Contexts of several documents in the 8-bit cache, odd tree sizes.
        _tree("tree 8 users e4m3", 8, 4000, 32768, 15, 47, 12, 2, 128, "e4m3", "fp16", 32),
        # A full batch of a large model, wide trees.
        _tree("tree 32 users 64 drafts e4m3", 32, 1000, 8192, 64, 64, 32, 8, 128, "e4m3", "bf16"),
        # The rows of one decode step go into the cache.
        _rows("write 33 rows", "write", 33, 2, 128, "fp16"),
        # Prompt rows, columns of the fused projection of a large model.
        _rows("write 32768 rows", "write", 32768, 8, 128, "bf16", fused=32),
        # A short prefix read back by a program that works in 32 bits.
        _rows("read 500 rows", "read", 500, 2, 64, "f32"),
        # A long prefix of a large model read back for a prompt's attention.
        _rows("read 32768 rows", "read", 32768, 8, 128, "bf16", 32),
        # 24 drafted tokens of a small model, in 32 bits.
        _norm("norm 24 drafts", 24, 14, 2, 64, 64, 1, "f32", False, 4096),
        # Image and video patches: time, height and width, pairs side by side.
        _norm("norm patches of three axes", 8190, 12, 2, 128, 128, 3, "fp16", True, 1000),
        # A full batch of prompt rows of a large model.
        _norm("norm 32768 rows", 32768, 32, 8, 128, 128, 1, "bf16", False, 131072),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    what = rng.choice(["tree", "tree", "tree", "write", "read", "norm", "norm"])
    block = rng.choice([16, 16, 32, 48, 64])
    if what == "tree":
        hq, hkv, d = rng.choice([(14, 2, 64), (12, 2, 128), (32, 8, 128), (8, 1, 128), (16, 16, 96),
                                 (8, 1, 256), (24, 4, 32), (10, 2, 160)])
        seqs = _log(rng, 1, 64)
        most = min(rng.choice([1, 4, 8, 16, 32, 64, 64, 200]), 2048 // seqs)
        hi = max(_log(rng, 128, (16384 if most > 64 else 65536) // seqs), most)
        pool = rng.choice(["fp16", "e4m3", "e4m3"])
        c = _tree("", seqs, max(most, hi // rng.choice([1, 4, 16])), hi, rng.randint(1, most), most,
                  hq, hkv, d, pool, "fp16" if pool == "fp16" else rng.choice(["fp16", "bf16"]), block,
                  rng.randint(2, 1 << 20))
    elif what == "norm":
        hq, hkv, d = rng.choice([(14, 2, 64), (12, 2, 128), (32, 8, 128), (16, 16, 96), (8, 1, 256),
                                 (10, 2, 80)])
        c = _norm("", _log(rng, 1, 16384), hq, hkv, d, rng.choice([d, d, d // 2, 2 * rng.randint(1, d // 2)]),
                  rng.choice([1, 2, 3, 4]), rng.choice(["fp16", "bf16", "f32"]), rng.random() < 0.5,
                  _log(rng, 100, 1000000), rng.random() < 0.8)
    else:
        hkv, d = rng.choice([(2, 64), (2, 128), (8, 128), (16, 96), (1, 256), (4, 32), (2, 160)])
        types = ["fp16", "bf16"] if what == "write" else ["fp16", "bf16", "f32"]
        c = _rows("", what, _log(rng, 1, 16384), hkv, d, rng.choice(types), block,
                  rng.choice([0, 0, 4 * hkv]))
    del c["name"]
    return c


# ---------------------------------------------------------------------------- what a case holds
def _shape(case):
    """Drafted tokens and whole context of every sequence, and the parent of every drafted token."""
    r = np.random.default_rng(case["ragged"])
    new = r.integers(case["least"], case["most"] + 1, case["seqs"])
    ctx = np.exp(r.uniform(math.log(case["lo"]), math.log(case["hi"]), case["seqs"]))
    ctx = np.maximum(np.rint(ctx).astype(np.int64).clip(case["lo"], case["hi"]), new)
    # token 0 hangs on the context, every other one on an earlier one, mostly a late one
    at = np.arange(case["most"])
    parent = np.floor(at * r.random((case["seqs"], case["most"])) ** 0.5).astype(np.int64)
    parent[:, 0] = -1
    return new, ctx, parent


def _ancestors(parent):
    """[seqs][tokens][tokens]: 1 where the column's token is the row's own or an ancestor of it.
    (With P the parents, the sum of all powers of P is the inverse of 1 - P.)"""
    n = parent.shape[1]
    link = np.zeros(parent.shape + (n,))
    np.put_along_axis(link, np.maximum(parent, 0)[..., None], 1.0, 2)
    link[:, 0] = 0.0
    return np.linalg.inv(np.eye(n) - link) > 0.5


def _words(seen):
    """... as bits of 64-bit words."""
    n = seen.shape[2]
    words = (n + 63) // 64
    bits = np.zeros(seen.shape[:2] + (64 * words,), np.uint8)
    bits[..., :n] = seen
    return np.packbits(bits, axis=2, bitorder="little").view(np.int64)


def _normal(gen, *shape, dev=1.0):
    return torch.empty(*shape, device="cuda").normal_(0, dev, generator=gen)


def _cuda(a, dtype):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, dtype))).cuda()


def _ptr(t):
    return C.c_void_p(t.data_ptr())


def _quantised(x):
    """Head rows [..., d] in 32 bits -> e4m3 values as bytes, and the bytes of their exponents."""
    m, k = torch.frexp(x.abs().amax(-1))  # x = m 2^k, m in [0.5, 1); 448 = 0.875 2^9
    e = (k - 9 + (m > 0.875)).clamp(LOWEST, HIGHEST)
    e = torch.where(m == 0, LOWEST, e)
    codes = torch.ldexp(x, -e[..., None]).clamp(-448, 448).to(E4M3)
    return codes.view(torch.uint8), (e + 127).to(torch.uint8)


# ---------------------------------------------------------------------------- tree attention
def _tree_inputs(case, gen):
    new, ctx, parent = _shape(case)
    hq, hkv, d, b = case["hq"], case["hkv"], case["d"], case["block"]
    blocks = (ctx + b - 1) // b
    count = int(blocks.sum()) + 3
    q = _normal(gen, int(new.sum()), hq * d).to(TYPES[case["dtype"]])
    # some channels of K are larger than the others, as they are behind a projection
    channels = 1 + 3 * (torch.rand(hkv, d, device="cuda", generator=gen) < 0.05)
    k = (_normal(gen, count, b, hkv, d) * channels).to(torch.float16)
    v = _normal(gen, count, b, hkv, d, dev=0.5).to(torch.float16)
    table = np.zeros((case["seqs"], int(blocks.max())), np.int64)
    used = np.arange(table.shape[1])[None] < blocks[:, None]
    table[used] = np.random.default_rng(case["ragged"] + 1).permutation(count)[:int(blocks.sum())]
    return q, k, v, table


def _prepare_tree(case, gen):
    q, k, v, table = _tree_inputs(case, gen)
    new, ctx, parent = _shape(case)
    words = _words(_ancestors(parent))
    there = np.arange(case["most"])[None] < new[:, None]
    s = dict(case=case, q=q, out=torch.zeros_like(q), table=_cuda(table, np.int32), count=k.shape[0],
             cu=_cuda(np.concatenate([[0], np.cumsum(new)]), np.int32), ctx=_cuda(ctx, np.int32),
             mask=_cuda(words[there], np.int64), new=_cuda(new, np.int64), longest=int(new.max()))
    if case["pool"] == "e4m3":
        # (head rows are quantised; their exponents lie head by head within a block)
        s["k"], s["v"], s["k_exp"], s["v_exp"] = (
            *(_quantised(x.float())[0] for x in (k, v)),
            *(_quantised(x.float())[1].transpose(1, 2).contiguous() for x in (k, v)))
    else:
        s["k"], s["v"], s["k_exp"], s["v_exp"] = k, v, None, None
    if own:
        from logismos_amd import kernels
        s["ws"] = torch.empty(kernels.paged_attn_tree_workspace_bytes(
            q.shape[0], s["longest"], case["hq"], case["hkv"], case["d"]), dtype=torch.uint8,
            device="cuda")
    return s


def _plain_cache(pool, exp, table):
    """[seqs][keys][heads][d] in 32 bits of the blocks of a table."""
    x = pool[table]
    if exp is not None:
        x = torch.ldexp(x.view(E4M3).float(),
                        (exp[table].transpose(2, 3).int() - 127)[..., None])
    return x.float().flatten(1, 2)


def _plain_tree(s):
    c = s["case"]
    hq, hkv, d, S = c["hq"], c["hkv"], c["d"], c["seqs"]
    g, n = hq // hkv, s["longest"]
    table = s["table"].long()
    k = _plain_cache(s["k"], s["k_exp"], table).permute(0, 2, 3, 1).contiguous()
    v = _plain_cache(s["v"], s["v_exp"], table).transpose(1, 2).contiguous()
    # rows padded to the longest tree
    i = torch.arange(n, device="cuda")
    there = i < s["new"][:, None]
    row = (s["cu"][:-1, None] + i).clamp(max=s["q"].shape[0] - 1).long()
    q = s["q"].float()[row].view(S, n, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(S, hkv, n * g, d)
    score = (q @ k) * (1.0 / math.sqrt(d))
    key = torch.arange(k.shape[3], device="cuda")
    j = key - (s["ctx"].long() - s["new"])[:, None]
    bits = (s["mask"][row][..., None] >> torch.arange(64, device="cuda")).bitwise_and(1).flatten(2)
    far = bits.shape[2]
    own_bit = torch.take_along_dim(bits, j.clamp(0, far - 1)[:, None].expand(S, n, -1), 2) == 1
    seen = (j < 0)[:, None] | (own_bit & (j < s["new"][:, None])[:, None])
    score = score.view(S, hkv, n, g, -1).masked_fill_(~seen[:, None, :, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(S, hkv, n * g, -1)
    o = (p @ v).view(S, hkv, n, g, d).permute(0, 2, 1, 3, 4).reshape(S, n, hq * d)
    return o[there].to(s["q"].dtype)


def _own_tree(s):
    from logismos_amd import kernels
    c = s["case"]
    kernels.launch_paged_attn_tree(
        _ptr(s["q"]), _ptr(s["k"]), _ptr(s["v"]), _ptr(s["table"]), _ptr(s["cu"]), _ptr(s["ctx"]),
        _ptr(s["mask"]), _ptr(s["out"]), _ptr(s["ws"]), c["seqs"], s["q"].shape[0], s["longest"],
        c["hq"], c["hkv"], c["d"], c["block"], s["table"].shape[1], s["count"],
        1.0 / math.sqrt(c["d"]), mask_words=s["mask"].shape[1],
        k_exp=None if s["k_exp"] is None else _ptr(s["k_exp"]),
        v_exp=None if s["v_exp"] is None else _ptr(s["v_exp"]), bf16=c["dtype"] == "bf16")
    return s["out"]


def _exact_sequence(case, q, k, v, table, n, ctx, parent):
    hq, hkv, d, b = case["hq"], case["hkv"], case["d"], case["block"]
    ids = torch.from_numpy(table[:(ctx + b - 1) // b]).cuda()

    def rows(pool):
        x = pool[ids].reshape(-1, hkv, d)[:ctx].double()
        if case["pool"] == "e4m3":
            step = 2.0 ** torch.ceil(torch.log2(x.abs().amax(2, keepdim=True) / 448))
            x = (x / step).to(torch.float32).to(E4M3).double() * step
        return x.transpose(0, 1).contiguous()

    key, val = rows(k), rows(v)
    seen = np.zeros((n, ctx), bool)
    seen[:, :ctx - n] = True
    for i in range(n):
        seen[i, ctx - n + i] = True
        if parent[i] >= 0:
            seen[i] |= seen[parent[i]]
    hidden = torch.from_numpy(~seen).cuda()
    x = q.double().view(n, hkv, hq // hkv, d).transpose(0, 1).reshape(hkv, -1, d)
    logit = torch.bmm(x, key.transpose(1, 2).contiguous()) / math.sqrt(d)
    logit.view(hkv, n, -1, ctx).masked_fill_(hidden[None, :, None], -math.inf)
    o = torch.bmm(torch.softmax(logit, 2), val)
    return o.view(hkv, n, -1, d).transpose(0, 1).reshape(n, hq * d)


def _exact_tree(case, gen):
    q, k, v, table = _tree_inputs(case, gen)
    new, ctx, parent = _shape(case)
    ends = np.cumsum(new)
    return torch.cat([_exact_sequence(case, q[e - n:e], k, v, t, int(n), int(c), p)
                      for e, n, c, t, p in zip(ends, new, ctx, table, parent)])


def _work_tree(case):
    new, ctx, parent = _shape(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    seen = _ancestors(parent).sum(2) * (np.arange(case["most"])[None] < new[:, None])
    pairs = int((new * (ctx - new)).sum() + seen.sum())
    row = 2 * (d + 1) if case["pool"] == "e4m3" else 4 * d
    rows = int(new.sum())
    return dict(bytes=int(ctx.sum()) * hkv * row + 4 * rows * hq * d
                + 8 * rows * ((case["most"] + 63) // 64) + 8 * case["seqs"],
                flops=4 * pairs * hq * d)


# ---------------------------------------------------------------------------- the cache in 8 bits
def _columns(case, gen):
    """K and V rows: matrices of their own, or the last columns of fused rows of more heads."""
    hkv, d, T = case["hkv"], case["d"], case["tokens"]
    size = torch.exp2(_normal(gen, T, 1))  # tokens differ in size
    if case["fused"]:
        rows = (_normal(gen, T, (case["fused"] + 2 * hkv) * d) * size).to(TYPES[case["dtype"]])
        return rows[:, -2 * hkv * d:-hkv * d], rows[:, -hkv * d:]
    return tuple((_normal(gen, T, hkv * d) * size).to(TYPES[case["dtype"]]) for _ in range(2))


def _slots(case, gen):
    count = case["tokens"] // case["block"] + 2
    order = torch.randperm(count, device="cuda", generator=gen)
    at = torch.arange(case["tokens"], device="cuda")
    return order[at // case["block"]] * case["block"] + at % case["block"], count


def _prepare_write(case, gen):
    k, v = _columns(case, gen)
    slots, count = _slots(case, gen)
    b, hkv, d = case["block"], case["hkv"], case["d"]
    pool = [torch.zeros(count, b, hkv, d, dtype=torch.uint8, device="cuda") for _ in range(2)]
    exp = [torch.zeros(count, hkv, b, dtype=torch.uint8, device="cuda") for _ in range(2)]
    return dict(case=case, k=k, v=v, slots=slots, count=count, k_pool=pool[0], v_pool=pool[1],
                k_exp=exp[0], v_exp=exp[1])


def _cache(s):
    return dict(k=s["k_pool"].view(E4M3), v=s["v_pool"].view(E4M3), k_exp=s["k_exp"],
                v_exp=s["v_exp"])


def _plain_rows(x, pool, exp, s):
    c = s["case"]
    codes, e = _quantised(x.float().view(-1, c["hkv"], c["d"]))
    block, row = s["slots"] // c["block"], s["slots"] % c["block"]
    pool[block, row] = codes
    exp[block, :, row] = e


def _plain_write(s):
    _plain_rows(s["k"], s["k_pool"], s["k_exp"], s)
    _plain_rows(s["v"], s["v_pool"], s["v_exp"], s)
    return _cache(s)


def _own_write(s):
    from logismos_amd import kernels
    c = s["case"]
    kernels.launch_kv_write_e4m3(
        _ptr(s["k"]), _ptr(s["v"]), _ptr(s["k_pool"]), _ptr(s["k_exp"]), _ptr(s["v_pool"]),
        _ptr(s["v_exp"]), _ptr(s["slots"]), c["tokens"], c["hkv"], c["d"], c["block"], s["count"],
        k_stride=s["k"].stride(0), v_stride=s["v"].stride(0), bf16=c["dtype"] == "bf16")
    return _cache(s)


def _exact_write(case, gen):
    inputs = _columns(case, gen)
    slots, count = _slots(case, gen)
    b, hkv, d = case["block"], case["hkv"], case["d"]
    found = {}
    for name, x in zip("kv", inputs):
        x = x.double().reshape(-1, hkv, d)
        e = torch.ceil(torch.log2(x.abs().amax(2) / 448)).clamp(LOWEST, HIGHEST)
        pool = torch.zeros(count * b, hkv, d, dtype=torch.float64, device="cuda")
        pool[slots] = x * torch.exp2(-e)[..., None]
        exps = torch.zeros(count * b, hkv, dtype=torch.uint8, device="cuda")
        exps[slots] = (e + 127).to(torch.uint8)
        found[name] = pool.view(count, b, hkv, d)
        found[name + "_exp"] = exps.view(count, b, hkv).transpose(1, 2).contiguous()
    return dict(k=found["k"], v=found["v"], k_exp=found["k_exp"], v_exp=found["v_exp"])


def _prepare_read(case, gen):
    s = _prepare_write({**case, "dtype": "fp16", "fused": 0}, gen)
    _plain_write(s)
    shape = case["tokens"], case["hkv"] * case["d"]
    out = [torch.zeros(shape, dtype=TYPES[case["dtype"]], device="cuda") for _ in range(2)]
    return dict(case=case, slots=s["slots"], count=s["count"], k_pool=s["k_pool"], v_pool=s["v_pool"],
                k_exp=s["k_exp"], v_exp=s["v_exp"], k=out[0], v=out[1])


def _plain_back(pool, exp, s):
    c = s["case"]
    block, row = s["slots"] // c["block"], s["slots"] % c["block"]
    x = torch.ldexp(pool.view(E4M3)[block, row].float(), (exp[block, :, row].int() - 127)[..., None])
    return x.flatten(1).to(TYPES[c["dtype"]])


def _plain_read(s):
    return dict(k=_plain_back(s["k_pool"], s["k_exp"], s), v=_plain_back(s["v_pool"], s["v_exp"], s))


def _own_read(s):
    from logismos_amd import kernels
    c = s["case"]
    kernels.launch_kv_gather_e4m3(
        _ptr(s["k_pool"]), _ptr(s["k_exp"]), _ptr(s["v_pool"]), _ptr(s["v_exp"]), _ptr(s["slots"]),
        _ptr(s["k"]), _ptr(s["v"]), c["tokens"], c["hkv"], c["d"], c["block"], s["count"],
        dtype=c["dtype"])
    return dict(k=s["k"], v=s["v"])


def _exact_read(case, gen):
    inputs = _columns({**case, "dtype": "fp16", "fused": 0}, gen)
    found = {}
    for name, x in zip("kv", inputs):
        x = x.double().reshape(-1, case["hkv"], case["d"])
        step = torch.exp2(torch.ceil(torch.log2(x.abs().amax(2, keepdim=True) / 448)))
        found[name] = ((x / step).to(torch.float32).to(E4M3).double() * step).flatten(1)
    return found


def _work_rows(case):
    size = 4 if case["dtype"] == "f32" else 2
    values = 2 * case["tokens"] * case["hkv"] * case["d"]
    return dict(bytes=values * (size + 1) + 2 * case["tokens"] * case["hkv"] + 8 * case["tokens"],
                flops=2 * values)


# ---------------------------------------------------------------------------- norms and positions
def _norm_inputs(case, gen):
    T, d = case["tokens"], case["d"]
    rows = _normal(gen, T, (case["hq"] + 2 * case["hkv"]) * d, dev=2.0).to(TYPES[case["dtype"]])
    gains = 1 + _normal(gen, 2, d, dev=0.2)
    positions = torch.randint(case["far"], (case["axes"], T), generator=gen, device="cuda",
                              dtype=torch.int32)
    # the pairs of an axis lie side by side, the first axis has a few more
    pairs = case["rotary"] // 2
    axis = np.arange(pairs) * case["axes"] // max(pairs, 1)
    return rows, gains, positions, axis


def _prepare_norm(case, gen):
    rows, gains, positions, axis = _norm_inputs(case, gen)
    T, d = case["tokens"], case["d"]
    pairs = np.arange(case["rotary"] // 2)
    return dict(case=case, rows=rows, gains=gains, positions=positions, axis=_cuda(axis, np.uint8),
                f=_cuda(1e6 ** (-2.0 * pairs / case["rotary"]), np.float64),
                q=torch.zeros(T, case["hq"] * d, dtype=rows.dtype, device="cuda"),
                k=torch.zeros(T, case["hkv"] * d, dtype=rows.dtype, device="cuda"))


def _plain_norm(s):
    c = s["case"]
    d, r, hq, hkv = c["d"], c["rotary"], c["hq"], c["hkv"]
    angle = torch.remainder(s["positions"].double()[s["axis"].long()].t() * s["f"],
                            2 * math.pi).float()
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    x = s["rows"][:, :(hq + hkv) * d].float().reshape(c["tokens"], hq + hkv, d)
    if c["gains"]:
        head_gains = s["gains"].repeat_interleave(torch.tensor([hq, hkv], device="cuda"), 0,
                                                  output_size=hq + hkv)
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * head_gains
    one, two = (x[..., 0:r:2], x[..., 1:r:2]) if c["interleaved"] else \
        (x[..., :r // 2], x[..., r // 2:r])
    a, b = one * cos - two * sin, one * sin + two * cos
    turned = torch.stack([a, b], -1).flatten(-2) if c["interleaved"] else torch.cat([a, b], -1)
    y = torch.cat([turned, x[..., r:]], -1).to(s["rows"].dtype).flatten(1)
    return dict(q=y[:, :hq * d].contiguous(), k=y[:, hq * d:].contiguous())


def _own_norm(s):
    from logismos_amd import kernels
    c = s["case"]
    width, hq, d = s["rows"].shape[1], c["hq"], c["d"]
    kernels.launch_norm_rope_packed(
        _ptr(s["rows"]), _ptr(s["rows"][0, hq * d:]), _ptr(s["q"]), _ptr(s["k"]),
        _ptr(s["positions"]), _ptr(s["axis"]), _ptr(s["f"]),
        _ptr(s["gains"][0]) if c["gains"] else None, _ptr(s["gains"][1]) if c["gains"] else None,
        c["tokens"], hq, c["hkv"], d, c["rotary"], num_axes=c["axes"], eps=1e-6,
        interleaved=c["interleaved"], q_in_stride=width, k_in_stride=width, dtype=c["dtype"])
    return dict(q=s["q"], k=s["k"])


def _exact_norm(case, gen):
    rows, gains, positions, axis = _norm_inputs(case, gen)
    d, r, hq, heads = case["d"], case["rotary"], case["hq"], case["hq"] + case["hkv"]
    y = rows[:, :heads * d].double().reshape(-1, heads, d).clone()
    if case["gains"]:
        y /= torch.sqrt(y.square().sum(2, keepdim=True) / d + 1e-6)
        y[:, :hq] *= gains[0].double()
        y[:, hq:] *= gains[1].double()
    for i in range(r // 2):
        t = positions[int(axis[i])].double() * math.exp(-2 * i / r * math.log(1e6))
        p, q = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + r // 2)
        c, s_ = torch.cos(t)[:, None], torch.sin(t)[:, None]
        a, b = y[..., p].clone(), y[..., q].clone()
        y[..., p] = c * a - s_ * b
        y[..., q] = s_ * a + c * b
    y = y.reshape(-1, heads * d)
    return dict(q=y[:, :hq * d].contiguous(), k=y[:, hq * d:].contiguous())


def _work_norm(case):
    size = 4 if case["dtype"] == "f32" else 2
    T, heads, d = case["tokens"], case["hq"] + case["hkv"], case["d"]
    norm = 4 * d if case["gains"] else 0
    return dict(bytes=2 * size * T * heads * d + 4 * T * case["axes"] + 5 * case["rotary"] + 8 * d,
                flops=T * heads * (3 * case["rotary"] + norm))


# ----------------------------------------------------------------------------
def _gen(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def prepare(case, seed):
    return dict(tree=_prepare_tree, write=_prepare_write, read=_prepare_read,
                norm=_prepare_norm)[case["kind"]](case, _gen(seed))


def run(state):
    kind = state["case"]["kind"]
    if own:
        return dict(tree=_own_tree, write=_own_write, read=_own_read, norm=_own_norm)[kind](state)
    return dict(tree=_plain_tree, write=_plain_write, read=_plain_read, norm=_plain_norm)[kind](state)


def work(case):
    return dict(tree=_work_tree, write=_work_rows, read=_work_rows,
                norm=_work_norm)[case["kind"]](case)


def exact(case, seed):
    return dict(tree=_exact_tree, write=_exact_write, read=_exact_read,
                norm=_exact_norm)[case["kind"]](case, _gen(seed))
