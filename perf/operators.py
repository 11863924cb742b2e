"""The operators of the 8-bit paged key/value cache, as cases that can be timed.

Two kinds of work, through the public entry points of cublade_amd.quantization:

  append   append_kv (position rotation of keys and queries, quantisation of
           keys and values into their pages), then dequantize_kv of the pages
           that the call touched
  attend   attend_kv: attention of new queries over the cached keys and values

Where ``own`` is false, ``run`` computes the same from elementary torch
operations in 32 bits on the same cache buffers; ``exact`` gives the result in
64 bits, from the definition.

The cache: K codes [page, kv head, token, d], V codes [page, kv head, d,
token], one fp32 scale for each page and kv head. ``lengths`` counts a
sequence's tokens with the new ones, ``cu`` where each sequence's new tokens
start among all of them (None: one new token per sequence).
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
STORES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
QMAX = {"int8": 127.0, "fp8": 448.0}
EPS = 1e-12


def listed() -> list[dict]:
    return [
        # One user's decode step: one token into a partly filled page. Latency.
        dict(name="append_one", kind="append", b=1, n=1, n_lo=1, len_lo=700, len_hi=700, hq=32,
             hkv=8, d=128, rot=128, style="half", page=64, store="int8", dtype="bf16", window=0),
        # A decode step of many users, one cached head per query head, small pages.
        dict(name="append_batch", kind="append", b=256, n=1, n_lo=1, len_lo=1, len_hi=8000, hq=32,
             hkv=32, d=64, rot=64, style="interleaved", page=16, store="fp8", dtype="fp16",
             window=0),
        # A whole prompt entering an empty sequence.
        dict(name="append_prompt", kind="append", b=1, n=8192, n_lo=8192, len_lo=8192, len_hi=8192,
             hq=32, hkv=8, d=128, rot=128, style="half", page=64, store="int8", dtype="bf16",
             window=0),
        # Prompt chunks of several users, ragged, over pages already begun; only
        # half of each head is rotated.
        dict(name="append_ragged", kind="append", b=13, n=900, n_lo=1, len_lo=900, len_hi=5000,
             hq=24, hkv=6, d=96, rot=48, style="half", page=32, store="fp8", dtype="bf16",
             window=0),
        # The first tokens of a conversation. Latency.
        dict(name="attend_first", kind="attend", b=1, n=1, n_lo=1, len_lo=17, len_hi=17, hq=32,
             hkv=8, d=128, rot=128, style="half", page=64, store="int8", dtype="bf16", window=0),
        # One user with a very long context: few rows, a long axis.
        dict(name="attend_long", kind="attend", b=1, n=1, n_lo=1, len_lo=131077, len_hi=131077,
             hq=32, hkv=8, d=128, rot=128, style="half", page=64, store="int8", dtype="bf16",
             window=0),
        # A serving batch of mixed lengths, small pages, FP8 codes.
        dict(name="attend_batch", kind="attend", b=64, n=1, n_lo=1, len_lo=100, len_hi=8000, hq=32,
             hkv=8, d=128, rot=128, style="half", page=16, store="fp8", dtype="bf16", window=0),
        # A larger batch of a small model without shared heads.
        dict(name="attend_mha", kind="attend", b=128, n=1, n_lo=1, len_lo=900, len_hi=1100, hq=16,
             hkv=16, d=64, rot=64, style="half", page=32, store="int8", dtype="fp16", window=0),
        # Drafted tokens checked in one call: a few queries per sequence.
        dict(name="attend_draft", kind="attend", b=24, n=8, n_lo=1, len_lo=8, len_hi=4000, hq=40,
             hkv=8, d=128, rot=128, style="half", page=64, store="fp8", dtype="fp16", window=0),
        # A whole prompt at once.
        dict(name="attend_prompt", kind="attend", b=1, n=8192, n_lo=8192, len_lo=8192, len_hi=8192,
             hq=32, hkv=8, d=128, rot=128, style="half", page=64, store="int8", dtype="bf16",
             window=0),
        # One chunk of a long prompt, over what was cached before it.
        dict(name="attend_chunk", kind="attend", b=1, n=2048, n_lo=2048, len_lo=32768,
             len_hi=32768, hq=32, hkv=8, d=128, rot=128, style="half", page=128, store="fp8",
             dtype="fp16", window=0),
        # A mixed batch: single tokens of some users beside prompt chunks of
        # others, an odd head size, a sliding window.
        dict(name="attend_mixed", kind="attend", b=20, n=1500, n_lo=0, len_lo=1500, len_hi=6000,
             hq=16, hkv=4, d=80, rot=80, style="half", page=32, store="int8", dtype="bf16",
             window=1024),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    while True:
        hkv = rng.choice([1, 2, 4, 5, 8, 8, 16])
        d = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256])
        case = dict(kind=rng.choice(["append", "attend", "attend"]),
                    hq=hkv * rng.choice([1, 1, 2, 4, 4, 7, 8]), hkv=hkv, d=d,
                    rot=rng.choice([d, d, d // 2]), style=rng.choice(["half", "interleaved"]),
                    page=rng.choice([16, 32, 64, 64, 128]), store=rng.choice(["int8", "fp8"]),
                    dtype=rng.choice(["fp16", "bf16"]), window=0)
        form = rng.choice(["step", "step", "few", "prompt", "mixed"])
        if form == "step":
            b = _log_int(rng, 1, 256)
            hi = _log_int(rng, 1, 131072)
            case.update(b=b, n=1, n_lo=1, len_lo=max(1, int(hi * rng.uniform(0.05, 1))), len_hi=hi)
        elif form == "few":
            b, n = _log_int(rng, 1, 64), rng.randint(2, 16)
            hi = _log_int(rng, n, 32768)
            case.update(b=b, n=n, n_lo=1, len_lo=max(n, int(hi * rng.uniform(0.05, 1))), len_hi=hi)
        elif form == "prompt":
            n = _log_int(rng, 17, 8192)
            hi = max(n, _log_int(rng, n, 32768))
            case.update(b=rng.choice([1, 1, 2, 3]), n=n, n_lo=n, len_lo=hi, len_hi=hi)
        else:
            n = _log_int(rng, 64, 2048)
            case.update(b=rng.randint(3, 24), n=n, n_lo=0, len_lo=n, len_hi=_log_int(rng, n, 8192))
        if case["kind"] == "attend" and rng.random() < 0.2:
            case["window"] = _log_int(rng, 16, 4096)
        case["len_lo"] = min(case["len_lo"], case["len_hi"])
        # no more memory and no more work than the largest listed cases have
        cost = work(case)
        if (case["b"] * case["len_hi"] * case["hkv"] * d <= 64 * 8192 * 8 * 128
                and cost["flops"] <= 1.0e12 and cost["bytes"] <= 4.0e8):
            return case


# ---------------------------------------------------------------------------
# Sizes of a case: lengths and numbers of new tokens follow from its values
# ---------------------------------------------------------------------------
def _sizes(case: dict) -> tuple[list[int], list[int]]:
    """(lengths with the new tokens, new tokens) of every sequence. n_lo = 0
    stands for a mixed batch: three sequences in four bring one token."""
    rng = random.Random(f"{case['b']} {case['n']} {case['len_lo']} {case['len_hi']}")
    lens, news = [], []
    for i in range(case["b"]):
        if case["n_lo"] == 0:
            new = 1 if i % 4 else rng.randint(max(1, case["n"] // 8), case["n"])
        else:
            new = rng.randint(case["n_lo"], case["n"])
        lens.append(max(new, rng.randint(case["len_lo"], case["len_hi"])))
        news.append(new)
    return lens, news


def _pages_of(length: int, page: int) -> int:
    return -(-length // page)


def _touched(case: dict, lens, news) -> list[tuple[int, int]]:
    """(sequence, index of the page in it) of every page that gets new tokens."""
    page = case["page"]
    return [(i, p) for i, (ln, nw) in enumerate(zip(lens, news)) if nw
            for p in range((ln - nw) // page, _pages_of(ln, page))]


def work(case: dict) -> dict:
    lens, news = _sizes(case)
    hq, hkv, d, page, t = case["hq"], case["hkv"], case["d"], case["page"], sum(news)
    if case["kind"] == "append":
        touched = len(_touched(case, lens, news))
        # k, v and q in, q out, the new codes, the touched pages' codes and
        # scales, their values, the rows of the rotation tables
        b = 2 * 2 * t * hkv * d + 2 * 2 * t * hq * d + 2 * t * hkv * d
        b += touched * hkv * (2 * page * d * (1 + 2) + 8) + 4 * t * case["rot"]
        return {"bytes": b, "flops": 3 * t * (hq + hkv) * case["rot"] + 2 * t * hkv * d * 2}
    pairs = keys = 0
    for ln, nw in zip(lens, news):
        first = ln - nw
        if case["window"]:
            w = case["window"]
            pairs += sum(min(p + 1, w) for p in range(first, ln))
            keys += ln - max(0, first - w + 1)
        else:
            pairs += nw * first + nw * (nw + 1) // 2
            keys += ln
    return {"bytes": 2 * 2 * t * hq * d + 2 * keys * hkv * d + 8 * hkv * keys // page,
            "flops": 4 * hq * d * pairs}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def prepare(case: dict, seed: int) -> dict:
    """What a serving program holds before the call: the cache with its earlier
    tokens, page tables in the order an allocator gives pages out, lengths,
    rotation tables, and the layer's new q, k and v."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    lens, news = _sizes(case)
    hq, hkv, d, page, t = case["hq"], case["hkv"], case["d"], case["page"], sum(news)
    dt = DTYPES[case["dtype"]]

    need = [_pages_of(ln, page) for ln in lens]
    pages = sum(need) + 8
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(case["b"], max(need) + 3, dtype=torch.int32, device=DEV)
    at = 0
    for i, c in enumerate(need):
        table[i, :c] = order[at:at + c]
        at += c

    def codes(shape):
        out = torch.empty(shape, dtype=STORES[case["store"]], device=DEV)
        step = max(1, (1 << 27) // math.prod(shape[1:]))
        spread = QMAX[case["store"]] / 4
        for p in range(0, pages, step):
            x = torch.randn((min(step, pages - p),) + shape[1:], generator=g, device=DEV)
            x = (x * spread).clamp_(-QMAX[case["store"]], QMAX[case["store"]])
            out[p:p + step] = x.round_() if case["store"] == "int8" else x
        return out

    def scales():   # a page's largest value is about 4 standard deviations of one
        return (torch.rand(pages, hkv, generator=g, device=DEV) * 0.6 + 0.7) * (
            4 / QMAX[case["store"]])

    st = dict(case=case, lens=lens, news=news, table=table,
              lengths=torch.tensor(lens, dtype=torch.int32, device=DEV),
              k_codes=codes((pages, hkv, page, d)), v_codes=codes((pages, hkv, d, page)),
              k_scale=scales(), v_scale=scales(), cu=None)
    if case["n"] > 1:
        ends = [0]
        for nw in news:
            ends.append(ends[-1] + nw)
        st["cu"] = torch.tensor(ends, dtype=torch.int32, device=DEV)
    # the fused projection's output: q, k and v of a token side by side
    qkv = torch.randn(t, hq + 2 * hkv, d, generator=g, device=DEV)
    qkv[:, hq:hq + hkv] *= torch.rand(d, generator=g, device=DEV) + 0.5
    qkv[:, hq:] *= 1 + (torch.rand(t, 1, 1, generator=g, device=DEV) < 0.02).float()
    qkv = qkv.to(dt)
    st.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:])
    if case["kind"] == "attend":
        st["q"] = st["q"].contiguous()
    half = case["rot"] // 2
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
    ang = torch.arange(max(lens), dtype=torch.float64, device=DEV)[:, None] * freq
    st.update(cos=ang.cos().float(), sin=ang.sin().float())
    touched = _touched(case, lens, news)
    st["touched"] = table[torch.tensor([i for i, _ in touched], device=DEV),
                          torch.tensor([p for _, p in touched], device=DEV)]
    if own:
        from cublade_amd.quantization import QuantizedKVCache
        st["cache"] = QuantizedKVCache(st["k_codes"], st["v_codes"], st["k_scale"], st["v_scale"])
    return st


def run(st: dict):
    case = st["case"]
    if own:
        from cublade_amd.quantization import append_kv, attend_kv, dequantize_kv
        if case["kind"] == "append":
            q = append_kv(st["cache"], st["k"], st["v"], st["table"], st["lengths"], cu_new=st["cu"],
                          rope=(st["cos"], st["sin"]), interleaved=case["style"] == "interleaved",
                          q=st["q"])
            return [q, *dequantize_kv(st["cache"], st["touched"], DTYPES[case["dtype"]])]
        return [attend_kv(st["q"], st["cache"], st["table"], st["lengths"], cu_q=st["cu"],
                          window=case["window"] or None)]
    return _plain_append(st) if case["kind"] == "append" else _plain_attend(st)


# ---------------------------------------------------------------------------
# Plain forms: elementary torch operations in 32 bits
# ---------------------------------------------------------------------------
def _token_index(st: dict):
    """For every new token: its position, and its row among the touched pages."""
    case, pos, row, base = st["case"], [], [], 0
    for ln, nw in zip(st["lens"], st["news"]):
        first = ln - nw
        pos += range(first, ln)
        if nw:
            p0 = first // case["page"]
            row += [base + p // case["page"] - p0 for p in range(first, ln)]
            base += _pages_of(ln, case["page"]) - p0
    return (torch.tensor(pos, device=DEV), torch.tensor(row, device=DEV))


def _rotate(x, cos, sin, rot: int, style: str):
    x = x.float()
    c, s = cos[:, None, :], sin[:, None, :]
    if style == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], dim=-1)


def _encode(x, store: str):
    if store == "int8":
        return torch.round(x).clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _plain_store(st: dict, x, pos, row, codes, scale, token_axis: int):
    """Quantises the new tokens' values x [t, hkv, d] into their pages."""
    case, touched = st["case"], st["touched"].long()
    page, hkv, d, qmax = case["page"], case["hkv"], case["d"], QMAX[case["store"]]
    n = touched.numel()
    new = torch.zeros(n, page, hkv, d, device=DEV)
    fresh = torch.zeros(n, page, dtype=torch.bool, device=DEV)
    new[row, pos % page] = x
    fresh[row, pos % page] = True
    amax = new.abs().amax(dim=(1, 3))                                  # [n, hkv]
    start = torch.full((n,), page, device=DEV).scatter_reduce(0, row, pos % page, "amin")
    begun = (start > 0)[:, None]                                       # holds earlier tokens
    inv_new = torch.full_like(amax, qmax) / amax.clamp(min=EPS)        # one rounding
    s_old = scale[touched]
    mant, exp = torch.frexp(amax / (qmax * s_old))
    grow = torch.where(mant > 0.5, exp, exp - 1).clamp(min=0) * begun
    s_kept = torch.ldexp(s_old, grow)
    s = torch.where(begun, s_kept, 1 / inv_new)
    inv = torch.where(begun, 1 / s_kept, inv_new)
    old = codes[touched]
    if token_axis == 3:
        old = old.transpose(2, 3)                                      # [n, hkv, page, d]
    slot = torch.arange(page, device=DEV)
    earlier = (slot < start[:, None])[:, None, :, None]
    is_new = fresh[:, None, :, None]
    lowered = _encode(torch.ldexp(old.float(), -grow[:, :, None, None]), case["store"])
    fresh_codes = _encode(new.permute(0, 2, 1, 3) * inv[:, :, None, None], case["store"])
    out = torch.where(is_new, fresh_codes.float(), torch.where(earlier, lowered.float(), old.float()))
    value = out * s[:, :, None, None]
    out = out.to(codes.dtype)
    codes[touched] = out.transpose(2, 3) if token_axis == 3 else out
    scale[touched] = s
    return value.to(DTYPES[case["dtype"]])


def _plain_append(st: dict):
    case = st["case"]
    pos, row = _token_index(st)
    cos, sin = st["cos"][pos], st["sin"][pos]
    q = _rotate(st["q"], cos, sin, case["rot"], case["style"])
    k = _rotate(st["k"], cos, sin, case["rot"], case["style"])
    return [q.to(DTYPES[case["dtype"]]),
            _plain_store(st, k, pos, row, st["k_codes"], st["k_scale"], 2),
            _plain_store(st, st["v"].float(), pos, row, st["v_codes"], st["v_scale"], 3)]


def _plain_attend(st: dict):
    case = st["case"]
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    rep = hq // hkv
    out = torch.zeros(st["q"].shape, dtype=st["q"].dtype, device=DEV)
    at = 0
    for i, (ln, nw) in enumerate(zip(st["lens"], st["news"])):
        if nw == 0:
            continue
        lo = max(0, ln - nw - case["window"] + 1) // page if case["window"] else 0
        ids = st["table"][i, lo:_pages_of(ln, page)].long()
        first = lo * page
        k = st["k_codes"][ids].float() * st["k_scale"][ids][:, :, None, None]
        v = st["v_codes"][ids].float() * st["v_scale"][ids][:, :, None, None]
        k = k.transpose(0, 1).reshape(hkv, -1, d)[:, :ln - first]
        v = v.permute(1, 0, 3, 2).reshape(hkv, -1, d)[:, :ln - first]
        q = st["q"][at:at + nw].float() / math.sqrt(d)
        key = torch.arange(first, ln, device=DEV)
        query = torch.arange(ln - nw, ln, device=DEV)
        hidden = key > query[:, None]
        if case["window"]:
            hidden |= key <= query[:, None] - case["window"]
        for h in range(hkv):
            s = (q[:, h * rep:(h + 1) * rep].transpose(0, 1).reshape(rep * nw, d) @ k[h].t())
            s = s.view(rep, nw, -1).masked_fill_(hidden, float("-inf"))
            p = (s - s.amax(-1, keepdim=True)).exp_()
            o = (p.view(rep * nw, -1) @ v[h]).view(rep, nw, d) / p.sum(-1, keepdim=True)
            out[at:at + nw, h * rep:(h + 1) * rep] = o.transpose(0, 1)
        at += nw
    return [out]


# ---------------------------------------------------------------------------
# The results in 64 bits
# ---------------------------------------------------------------------------
def _exact_code(x, store: str):
    """The value that the code nearest to x stands for (ties to even)."""
    if store == "int8":
        return x.round().clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return ((x / step).round() * step).clamp(-448, 448)


def _exact_turn(vec, pos: int, st: dict):
    """vec [heads, d] in 64 bits, turned to position pos: each pair is a complex
    number multiplied by cos + i sin."""
    rot = st["case"]["rot"]
    out = vec.clone()
    turn = torch.complex(st["cos"][pos].double(), st["sin"][pos].double())
    if st["case"]["style"] == "half":
        i1, i2 = slice(0, rot // 2), slice(rot // 2, rot)
    else:
        i1, i2 = slice(0, rot, 2), slice(1, rot, 2)
    z = torch.complex(vec[..., i1].contiguous(), vec[..., i2].contiguous()) * turn
    out[..., i1], out[..., i2] = z.real, z.imag
    return out


def exact(case: dict, seed: int):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    page, store = case["page"], case["store"]
    rep, qmax = case["hq"] // case["hkv"], QMAX[case["store"]]
    if case["kind"] == "append":
        q_out, ks, vs, at = [], [], [], 0
        for i, (ln, nw) in enumerate(zip(st["lens"], st["news"])):
            first = ln - nw
            for p in range(first // page, _pages_of(ln, page) if nw else 0):
                a, b = max(first, p * page), min(ln, (p + 1) * page)
                tok = slice(at + a - first, at + b - first)
                pos = torch.arange(a, b, device=DEV)[:, None]
                q_out.append(_exact_turn(st["q"][tok].double(), pos, st))
                pid = int(st["table"][i, p])
                for new, codes, scale, res in (
                        (_exact_turn(st["k"][tok].double(), pos, st), st["k_codes"][pid],
                         st["k_scale"][pid], ks),
                        (st["v"][tok].double(), st["v_codes"][pid].transpose(1, 2),
                         st["v_scale"][pid], vs)):
                    new = new.transpose(0, 1)                          # [hkv, tokens, d]
                    old, s = codes.double(), scale.double()
                    amax = new.abs().amax(dim=(1, 2))
                    n_old = a - p * page
                    if n_old == 0:
                        s = amax.clamp(min=EPS) / qmax
                    else:
                        g = torch.ceil(torch.log2(amax / (qmax * s))).clamp(min=0)
                        s = s * torch.exp2(g)
                        old[:, :n_old] = _exact_code(old[:, :n_old] * torch.exp2(-g)[:, None, None],
                                                     store)
                    old[:, n_old:n_old + b - a] = _exact_code(new / s[:, None, None], store)
                    res.append(old * s[:, None, None])
            at += nw
        return [torch.cat(q_out), torch.stack(ks), torch.stack(vs)]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    at = 0
    for i, (ln, nw) in enumerate(zip(st["lens"], st["news"])):
        ids = st["table"][i, :_pages_of(ln, page)].long()
        where = torch.arange(ln, device=DEV)
        for h in range(case["hkv"] if nw else 0):
            k = (st["k_codes"][ids, h].double() * st["k_scale"][ids, h].double()[:, None, None])
            v = (st["v_codes"][ids, h].double() * st["v_scale"][ids, h].double()[:, None, None])
            k, v = k.flatten(0, 1)[:ln], v.transpose(1, 2).flatten(0, 1)[:ln]
            for r in range(h * rep, (h + 1) * rep):
                for t0 in range(0, nw, 1024):
                    t1 = min(nw, t0 + 1024)
                    p = torch.arange(ln - nw + t0, ln - nw + t1, device=DEV)[:, None]
                    seen = where <= p
                    if case["window"]:
                        seen &= where > p - case["window"]
                    s = st["q"][at + t0:at + t1, r].double() @ k.t() * case["d"] ** -0.5
                    s[~seen] = float("-inf")
                    out[at + t0:at + t1, r] = torch.softmax(s, dim=-1) @ v
        at += nw
    return [out]
