"""The operators of an attention block over packed rows, as timed cases.

Three operators, in the order in which such a block calls them behind a shared projection:

* `adapter`: what the low-rank adapter of each request adds to the projection's rows,
  `out = base + scale_a * (x A_a^T) B_a^T`;
* `rope`: rotary positions of the q and k columns of fused q/k/v rows, in both layouts, over the
  whole head or its first part, with frequencies scaled for long contexts;
* `attn`: attention of whole packed sequences (prompts: causal; documents of an encoder:
  bidirectional), several query heads per KV head.

Head counts, widths and lengths are those of the repository's own geometries: 14 query and 2 KV
heads of 64, 12 and 2 of 128, 32 and 8 of 128, with rows of 896, 1536 and 4096.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
NONE, LINEAR, BASE, PARTS = 0, 1, 2, 3  # how the frequencies of rotary positions are scaled


def _attn(name, lo, hi, seqs, hq, hkv, d, dtype, causal, fused=True, ragged=1):
    return dict(name=name, kind="attn", lo=lo, hi=hi, seqs=seqs, hq=hq, hkv=hkv, d=d, dtype=dtype,
                causal=causal, fused=fused, ragged=ragged)


def _rope(name, tokens, hq, hkv, d, rotary, dtype, interleaved, far, scaling=NONE, factor=1.0,
          original=32768):
    return dict(name=name, kind="rope", tokens=tokens, hq=hq, hkv=hkv, d=d, rotary=rotary,
                dtype=dtype, interleaved=interleaved, far=far, scaling=scaling, factor=factor,
                original=original)


def _adapter(name, single, chunks, lo, hi, adapters, max_rank, n, k, dtype, f32_out=False, bare=0.0,
             ragged=1):
    return dict(name=name, kind="adapter", single=single, chunks=chunks, lo=lo, hi=hi,
                adapters=adapters, max_rank=max_rank, n=n, k=k, dtype=dtype, f32_out=f32_out,
                bare=bare, ragged=ragged)


def listed():
    return [
        # A search query on its way through an encoder: the smallest call.
        _attn("attn one query of 24", 24, 24, 1, 12, 2, 128, "fp16", False),
        # A batch of documents of an encoder, lengths as they come.
        _attn("attn 48 documents", 16, 512, 48, 12, 2, 128, "fp16", False),
        # Prompts of a small model with heads of 64.
        _attn("attn 8 prompts heads of 64", 100, 4096, 8, 14, 2, 64, "bf16", True),
        # One long prompt of a large model.
        _attn("attn prompt of 16384", 16384, 16384, 1, 32, 8, 128, "bf16", True),
        # The next tokens of 32 conversations.
        _rope("rope 32 users", 32, 32, 8, 128, 128, "bf16", False, 8192),
        # Encoder rows, pairs side by side.
        _rope("rope documents interleaved", 2036, 12, 2, 128, 128, "fp16", True, 509),
        # Half of each head rotated, far beyond the trained length.
        _rope("rope half the head by parts", 16384, 32, 8, 128, 64, "bf16", False, 500000, PARTS,
              16.0),
        # A full batch of prompt rows of a large model.
        _rope("rope 32768 rows linear", 32768, 32, 8, 128, 128, "bf16", False, 131072, LINEAR, 4.0),
        # One user with an adapter of his own.
        _adapter("adapter 1 user", 1, 0, 1, 1, 1, 16, 4096, 4096, "bf16"),
        # 32 conversations on 8 adapters of different ranks, a few on none: the q/k/v projection.
        _adapter("adapter 32 users", 32, 0, 1, 1, 8, 64, 6144, 4096, "bf16", bare=0.2),
        # Prompts of odd lengths next to single tokens: the down projection of a small model, its
        # sums kept in 32 bits.
        _adapter("adapter mixed batch", 13, 5, 31, 600, 6, 32, 1536, 8960, "fp16", f32_out=True,
                 bare=0.1),
        # 16 prompts of 512 through the gate/up projection of the large model.
        _adapter("adapter 16 prompts", 0, 16, 512, 512, 16, 64, 24576, 4096, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    what = rng.choice(["attn", "attn", "rope", "adapter", "adapter"])
    if what == "attn":
        hq, hkv, d = rng.choice([(14, 2, 64), (12, 2, 128), (32, 8, 128), (16, 16, 64), (8, 1, 128),
                                 (16, 16, 96), (8, 2, 256), (24, 4, 32)])
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 1, 8192 // seqs)
        c = _attn("", max(1, hi // rng.choice([1, 4, 16])), hi, seqs, hq, hkv, d,
                  rng.choice(["fp16", "bf16"]), rng.random() < 0.6, rng.random() < 0.7,
                  rng.randint(2, 1 << 20))
    elif what == "rope":
        hq, hkv, d = rng.choice([(14, 2, 64), (12, 2, 128), (32, 8, 128), (16, 16, 64), (16, 16, 96),
                                 (8, 2, 256)])
        rotary = rng.choice([d, d, d // 2, 2 * rng.randint(1, d // 2)])
        c = _rope("", _log(rng, 1, 16384), hq, hkv, d, rotary, rng.choice(["fp16", "bf16", "f32"]),
                  rng.random() < 0.5, _log(rng, 100, 1000000),
                  rng.choice([NONE, LINEAR, BASE, PARTS] if rotary > 2 else [NONE, LINEAR, PARTS]),
                  rng.uniform(1, 32), rng.choice([2048, 4096, 32768]))
    else:
        hidden = rng.choice([896, 1536, 4096])
        n = rng.choice([hidden, 8 * _log(rng, 64, 1536)])
        c = _adapter("", _log(rng, 1, 64), rng.choice([0, _log(rng, 1, 8)]), 1, _log(rng, 2, 512),
                     _log(rng, 1, 32), 8 * rng.choice([1, 2, 3, 4, 8, 16]), n,
                     8 * _log(rng, 112, 1120), rng.choice(["fp16", "bf16"]), rng.random() < 0.3,
                     rng.choice([0.0, 0.3]), rng.randint(2, 1 << 20))
    del c["name"]
    return c


# ---------------------------------------------------------------------------- what a case holds
def _lengths(case):
    """Tokens of every sequence, from the case's own numbers."""
    r = np.random.default_rng(case["ragged"])
    if case["kind"] == "attn":
        n = np.exp(r.uniform(math.log(case["lo"]), math.log(case["hi"]), case["seqs"]))
        return np.rint(n).astype(np.int64).clip(case["lo"], case["hi"])
    n = np.concatenate([np.ones(case["single"], np.int64),
                        r.integers(case["lo"], case["hi"] + 1, case["chunks"])])
    return n[r.permutation(len(n))]


def _choice(case):
    """Adapter of every sequence (-1: none) and rank of every adapter."""
    r = np.random.default_rng(case["ragged"] + 1)
    seqs = case["single"] + case["chunks"]
    pick = r.integers(0, case["adapters"], seqs)
    pick[r.random(seqs) < case["bare"]] = -1
    top = case["max_rank"]
    ranks = r.integers(max(1, top // 4), top + 1, case["adapters"])
    ranks[0] = top
    return pick, ranks


def _normal(gen, *shape, dev=1.0):
    return torch.empty(*shape, device="cuda").normal_(0, dev, generator=gen)


def _int32(a):
    return torch.from_numpy(np.asarray(a, np.int32)).cuda()


def _ptr(t, elements=0):
    return C.c_void_p(t.data_ptr() + elements * t.element_size())


# ---------------------------------------------------------------------------- attention
def _attn_inputs(case, gen):
    T, dtype = int(_lengths(case).sum()), TYPES[case["dtype"]]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["fused"]:
        rows = _normal(gen, T, (hq + 2 * hkv) * d).to(dtype)
        q, k, v = rows.split([hq * d, hkv * d, hkv * d], 1)
    else:
        q, k, v = (_normal(gen, T, h * d).to(dtype) for h in (hq, hkv, hkv))
    return q, k, v


def _prepare_attn(case, gen):
    q, k, v = _attn_inputs(case, gen)
    lens = _lengths(case)
    return dict(case=case, q=q, k=k, v=v, lens=lens.tolist(),
                cu=_int32(np.concatenate([[0], np.cumsum(lens)])),
                out=torch.zeros(q.shape, dtype=q.dtype, device="cuda"))


def _plain_attn(s):
    c = s["case"]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    g, scale = hq // hkv, 1.0 / math.sqrt(d)
    out = torch.empty(s["q"].shape, dtype=s["q"].dtype, device="cuda")
    at = 0
    for n in s["lens"]:
        rows = slice(at, at + n)
        q = s["q"][rows].float().view(n, hkv, g, d)
        k, v = s["k"][rows].float().view(n, hkv, d), s["v"][rows].float().view(n, hkv, d)
        for h in range(hkv):
            kh, vh = k[:, h].t().contiguous(), v[:, h].contiguous()
            for i in range(0, n, 4096):
                m = min(4096, n - i)
                scores = (q[i:i + m, h].reshape(m * g, d) @ kh) * scale
                if c["causal"]:
                    row = torch.arange(i, i + m, device="cuda").repeat_interleave(g)
                    scores.masked_fill_(torch.arange(n, device="cuda")[None] > row[:, None],
                                        -math.inf)
                p = torch.exp(scores - scores.amax(1, keepdim=True))
                o = (p @ vh) / p.sum(1, keepdim=True)
                out[at + i:at + i + m, h * g * d:(h + 1) * g * d] = o.view(m, g * d)
        at += n
    return out


def _own_attn(s):
    from logismos_amd import kernels
    c = s["case"]
    kernels.launch_attn_packed(
        _ptr(s["q"]), _ptr(s["k"]), _ptr(s["v"]), _ptr(s["cu"]), _ptr(s["out"]), len(s["lens"]),
        s["q"].shape[0], c["hq"], c["hkv"], c["d"], 1.0 / math.sqrt(c["d"]), causal=c["causal"],
        q_stride=s["q"].stride(0), k_stride=s["k"].stride(0), v_stride=s["v"].stride(0),
        bf16=c["dtype"] == "bf16")
    return s["out"]


def _exact_attn(case, gen):
    q, k, v = _attn_inputs(case, gen)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    lens = _lengths(case)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    ends = np.cumsum(lens)
    for head in range(hq):
        qs, ks = slice(head * d, (head + 1) * d), slice(head // (hq // hkv) * d,
                                                       (head // (hq // hkv) + 1) * d)
        for n, e in zip(lens.tolist(), ends.tolist()):
            key, val = k[e - n:e, ks].double(), v[e - n:e, ks].double().contiguous()
            for i in range(0, n, 2048):
                j = min(n, i + 2048)
                last = j if case["causal"] else n
                logit = q[e - n + i:e - n + j, qs].double() @ key[:last].t().contiguous()
                logit /= math.sqrt(d)
                if case["causal"]:
                    logit += torch.full((j - i, last), -math.inf, dtype=torch.float64,
                                        device="cuda").triu_(i + 1)
                out[e - n + i:e - n + j, qs] = torch.softmax(logit, 1) @ val[:last]
    return out


def _work_attn(case):
    lens = _lengths(case)
    T, d = int(lens.sum()), case["d"]
    pairs = int((lens * (lens + 1) // 2).sum() if case["causal"] else (lens * lens).sum())
    return dict(bytes=2 * T * d * 2 * (case["hq"] + case["hkv"]) + 4 * (len(lens) + 1),
                flops=4 * pairs * case["hq"] * d)


# ---------------------------------------------------------------------------- rotary positions
def _rope_inputs(case, gen):
    T, d = case["tokens"], case["d"]
    rows = _normal(gen, T, (case["hq"] + 2 * case["hkv"]) * d).to(TYPES[case["dtype"]])
    positions = torch.randint(case["far"], (T,), generator=gen, device="cuda", dtype=torch.int32)
    return rows, positions


def _plain_frequencies(case):
    """Radians per position of every rotated pair in 64 bits, and what cos and sin are times."""
    r, s, base = case["rotary"], case["factor"], 1e6
    if case["scaling"] == BASE:
        base *= s ** (r / (r - 2))
    f = base ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r)
    if case["scaling"] == LINEAR:
        f = f / s
    if case["scaling"] == PARTS:
        keep = ((case["original"] * f / (2 * math.pi) - 1) / (32 - 1)).clamp(0, 1)
        return keep * f + (1 - keep) * f / s, 0.1 * math.log(s) + 1
    return f, 1.0


def _prepare_rope(case, gen):
    rows, positions = _rope_inputs(case, gen)
    T, d = case["tokens"], case["d"]
    if own:
        from logismos_amd import kernels
        f, amplitude = kernels.rope_frequencies(
            case["rotary"], 1e6, scaling=("none", "linear", "base", "parts")[case["scaling"]],
            factor=case["factor"], original_positions=case["original"])
        f = torch.from_numpy(f).cuda()
    else:
        f, amplitude = _plain_frequencies(case)
    return dict(case=case, rows=rows, positions=positions, f=f, amplitude=amplitude,
                q=torch.zeros(T, case["hq"] * d, dtype=rows.dtype, device="cuda"),
                k=torch.zeros(T, case["hkv"] * d, dtype=rows.dtype, device="cuda"))


def _plain_rope(s):
    c = s["case"]
    d, r, hq, hkv = c["d"], c["rotary"], c["hq"], c["hkv"]
    angle = torch.remainder(s["positions"].double()[:, None] * s["f"], 2 * math.pi).float()
    cos = (angle.cos() * s["amplitude"])[:, None]
    sin = (angle.sin() * s["amplitude"])[:, None]
    x = s["rows"][:, :(hq + hkv) * d].float().reshape(c["tokens"], hq + hkv, d)
    one, two = (x[..., 0:r:2], x[..., 1:r:2]) if c["interleaved"] else \
        (x[..., :r // 2], x[..., r // 2:r])
    a, b = one * cos - two * sin, one * sin + two * cos
    turned = torch.stack([a, b], -1).flatten(-2) if c["interleaved"] else torch.cat([a, b], -1)
    y = torch.cat([turned, x[..., r:]], -1).to(s["rows"].dtype).flatten(1)
    return dict(q=y[:, :hq * d].contiguous(), k=y[:, hq * d:].contiguous())


def _own_rope(s):
    from logismos_amd import kernels
    c = s["case"]
    width = s["rows"].shape[1]
    kernels.launch_rope_packed(
        _ptr(s["rows"]), _ptr(s["rows"], c["hq"] * c["d"]), _ptr(s["q"]), _ptr(s["k"]),
        _ptr(s["positions"]), _ptr(s["f"]), c["tokens"], c["hq"], c["hkv"], c["d"], c["rotary"],
        interleaved=c["interleaved"], amplitude=s["amplitude"], q_in_stride=width,
        k_in_stride=width, dtype=c["dtype"])
    return dict(q=s["q"], k=s["k"])


def _exact_rope(case, gen):
    rows, positions = _rope_inputs(case, gen)
    r, d, s, heads = case["rotary"], case["d"], case["factor"], case["hq"] + case["hkv"]
    f, amplitude = [], 1.0
    for i in range(r // 2):
        theta = 1e6 * (s ** (r / (r - 2)) if case["scaling"] == BASE else 1.0)
        w = math.exp(-2 * i / r * math.log(theta))
        if case["scaling"] == LINEAR:
            w /= s
        elif case["scaling"] == PARTS:
            turns = case["original"] * w / (2 * math.pi)
            gamma = min(1.0, max(0.0, (turns - 1) / 31))
            w = w * gamma + w / s * (1 - gamma)
            amplitude = 0.1 * math.log(s) + 1
        f.append(w)
    y = rows[:, :heads * d].double().reshape(-1, heads, d).clone()
    at = positions.double()
    for i, w in enumerate(f):
        p, q = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + r // 2)
        c, s_ = (torch.cos(at * w) * amplitude)[:, None], (torch.sin(at * w) * amplitude)[:, None]
        a, b = y[..., p].clone(), y[..., q].clone()
        y[..., p] = c * a - s_ * b
        y[..., q] = s_ * a + c * b
    y = y.reshape(-1, heads * d)
    return dict(q=y[:, :case["hq"] * d].contiguous(), k=y[:, case["hq"] * d:].contiguous())


def _work_rope(case):
    size = 4 if case["dtype"] == "f32" else 2
    T, heads = case["tokens"], case["hq"] + case["hkv"]
    return dict(bytes=2 * size * T * heads * case["d"] + 4 * T + 4 * case["rotary"],
                flops=3 * T * heads * case["rotary"])


# ---------------------------------------------------------------------------- adapters
def _adapter_inputs(case, gen):
    T, dtype = int(_lengths(case).sum()), TYPES[case["dtype"]]
    n, k, r = case["n"], case["k"], case["max_rank"]
    x = _normal(gen, T, k).to(dtype)
    a = _normal(gen, case["adapters"], r, k, dev=1 / math.sqrt(k)).to(dtype)
    b = _normal(gen, case["adapters"], n, r, dev=0.05).to(dtype)
    base = _normal(gen, T, n).to(torch.float32 if case["f32_out"] else dtype)
    scales = 16.0 / torch.from_numpy(_choice(case)[1]).cuda().float()
    return x, a, b, base, scales


def _prepare_adapter(case, gen):
    x, a, b, base, scales = _adapter_inputs(case, gen)
    lens, (pick, ranks) = _lengths(case), _choice(case)
    s = dict(case=case, x=x, a=a, b=b, base=base, scales=scales, lens=lens.tolist(),
             pick_host=pick.tolist(), ranks_host=ranks.tolist(), scales_host=scales.tolist(),
             pick=_int32(pick), ranks=_int32(ranks),
             cu=_int32(np.concatenate([[0], np.cumsum(lens)])), out=torch.zeros_like(base))
    if own:
        from logismos_amd import kernels
        s["ws"] = torch.empty(kernels.adapter_add_workspace_bytes(x.shape[0], case["max_rank"]),
                              dtype=torch.uint8, device="cuda")
    return s


def _plain_adapter(s):
    out = s["base"].clone()
    at = 0
    for n, p in zip(s["lens"], s["pick_host"]):
        if p >= 0:
            r = s["ranks_host"][p]
            rows = slice(at, at + n)
            v = s["x"][rows].float() @ s["a"][p, :r].float().t()
            y = (v @ s["b"][p, :, :r].float().t()) * s["scales_host"][p]
            out[rows] = s["base"][rows].float() + y
        at += n
    return out


def _own_adapter(s):
    from logismos_amd import kernels
    c = s["case"]
    kernels.launch_adapter_add(
        _ptr(s["x"]), _ptr(s["a"]), _ptr(s["b"]), _ptr(s["ranks"]), _ptr(s["scales"]),
        _ptr(s["pick"]), _ptr(s["cu"]), _ptr(s["base"]), _ptr(s["out"]), _ptr(s["ws"]),
        len(s["lens"]), s["x"].shape[0], c["adapters"], c["max_rank"], c["n"], c["k"],
        bf16=c["dtype"] == "bf16", f32_out=c["f32_out"])
    return s["out"]


def _exact_adapter(case, gen):
    x, a, b, base, scales = _adapter_inputs(case, gen)
    pick, ranks = _choice(case)
    out = base.double()
    row_adapter = torch.from_numpy(np.repeat(pick, _lengths(case))).cuda()
    for p in range(case["adapters"]):
        rows = torch.nonzero(row_adapter == p).flatten()
        if len(rows):
            r = int(ranks[p])
            low = x[rows].double() @ a[p, :r].double().t().contiguous()
            out[rows] += float(scales[p]) * (low @ b[p, :, :r].double().t().contiguous())
    return out


def _work_adapter(case):
    lens, (pick, ranks) = _lengths(case), _choice(case)
    size = 4 if case["f32_out"] else 2
    used = sum(int(ranks[p]) for p in set(pick.tolist()) if p >= 0)
    rows = int(lens[pick >= 0].sum())
    flops = 2 * sum(int(n) * int(ranks[p]) for n, p in zip(lens, pick) if p >= 0) * \
        (case["n"] + case["k"])
    return dict(bytes=2 * used * (case["n"] + case["k"]) + 2 * rows * case["k"]
                + 2 * size * int(lens.sum()) * case["n"], flops=flops)


# ----------------------------------------------------------------------------
def _gen(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def prepare(case, seed):
    return dict(attn=_prepare_attn, rope=_prepare_rope,
                adapter=_prepare_adapter)[case["kind"]](case, _gen(seed))


def run(state):
    kind = state["case"]["kind"]
    if own:
        return dict(attn=_own_attn, rope=_own_rope, adapter=_own_adapter)[kind](state)
    return dict(attn=_plain_attn, rope=_plain_rope, adapter=_plain_adapter)[kind](state)


def work(case):
    return dict(attn=_work_attn, rope=_work_rope, adapter=_work_adapter)[case["kind"]](case)


def exact(case, seed):
    return dict(attn=_exact_attn, rope=_exact_rope,
                adapter=_exact_adapter)[case["kind"]](case, _gen(seed))
