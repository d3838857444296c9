"""Workloads of the operators between the projections and behind the LM head.

Three operators close a decode / verify step around the quantized linears:

* append -- norm of every query and key head, position rotation, and the append of keys and values to a paged cache;
* attend -- attention of a sequence's 1..16 newest tokens over that cache;
* sample -- one token per row of logits by temperature, top-k, top-p and min-p from a given uniform number.

`run` computes them in elementary torch operations (`own` false) or calls the library (`own` true); `exact` is their
definition in 64 bits.
"""
import ctypes as C
import os
import sys

import torch

own = False

_DEV = "cuda"
_CACHE = {"bf16": (torch.bfloat16, 0), "f16": (torch.float16, 1), "e4m3": (torch.float8_e4m3fn, 2)}
_EPS = 1e-6


# ---- the cases ------------------------------------------------------------------------------------------------------

def _append(name, tokens, heads, kv_heads, dim, rot, cache, act="f32", interleaved=False, page=64, gated=False):
    return {"name": name, "op": "append", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
            "cache": cache, "act": act, "interleaved": interleaved, "page": page, "gated": gated}


def _attend(name, seqs, new, kv_lo, kv_hi, heads, kv_heads, dim, cache, act="f32", page=64, ragged=False):
    return {"name": name, "op": "attend", "seqs": seqs, "new": new, "kv_lo": kv_lo, "kv_hi": kv_hi, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "cache": cache, "act": act, "page": page, "ragged": ragged}


def _sample(name, batch, vocab, temp, top_k, top_p, min_p, pad=0):
    return {"name": name, "op": "sample", "batch": batch, "vocab": vocab, "temp": temp, "top_k": top_k, "top_p": top_p,
            "min_p": min_p, "pad": pad}


def listed():
    return [
        # one decoded token of the model whose layer the benchmark measures: 24 query and 4 key heads of 256, 64 rotated
        _append("append_decode_1", 1, 24, 4, 256, 64, "bf16"),
        # verification of 8 tokens of each of 12 sequences, query heads interleaved with their output gates, 8-bit cache
        _append("append_verify_96", 96, 24, 4, 256, 64, "e4m3", gated=True),
        # a prefill chunk of the same model
        _append("append_prefill_2048", 2048, 24, 4, 256, 64, "bf16"),
        # a long prompt of an odd length in one piece, bf16 activations, heads of 128 rotated whole in neighbouring pairs
        _append("append_prefill_8191", 8191, 32, 8, 128, 128, "f16", act="bf16", interleaved=True, page=16),
        # one user, one token, a short conversation
        _attend("attend_1x2000", 1, 1, 2000, 2000, 24, 4, 256, "bf16"),
        # one user, one token, a context of 128 Ki tokens
        _attend("attend_1x131072", 1, 1, 131072, 131072, 24, 4, 256, "bf16", page=256),
        # speculative verification: 8 rows of each of 16 sequences, some with fewer drafts
        _attend("attend_verify_16x8", 16, 8, 1000, 8000, 24, 4, 256, "bf16", ragged=True),
        # a batch of users with contexts of all lengths (one slot idle), 8-bit cache
        _attend("attend_48_ragged_e4m3", 48, 1, 0, 16384, 24, 4, 256, "e4m3"),
        # a larger batch of a model with heads of 128, bf16 activations and fp16 cache
        _attend("attend_128x4096_f16", 128, 1, 4001, 4096, 32, 8, 128, "f16", act="bf16", page=16),
        # one user's token with the usual settings, over the vocabulary of the LM head the benchmark measures
        _sample("sample_1x248320", 1, 248320, 0.7, 20, 0.95, 0.0),
        # a batch that mixes settings row by row (greedy rows among them)
        _sample("sample_64x248320_mixed", 64, 248320, 0.0, 0, 0.0, 0.0),
        # temperature alone, an odd vocabulary with padded rows
        _sample("sample_8x32003_plain", 8, 32003, 1.0, 0, 1.0, 0.0, pad=13),
    ]


def _log(rng, lo, hi):
    import math
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


_HEADS = [(24, 4, 256), (16, 2, 256), (8, 8, 256), (32, 8, 128), (40, 8, 128), (28, 4, 128), (12, 12, 64), (20, 1, 64)]


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "sample"])
    cache = rng.choice(["bf16", "f16", "e4m3"])
    act = rng.choice(["f32", "f32", "bf16"])
    heads, kv_heads, dim = rng.choice(_HEADS)
    page = rng.choice([8, 16, 32, 48, 64, 128, 256])
    if op == "append":
        rot = rng.choice([dim, dim // 2, dim // 4])
        c = _append("", _log(rng, 1, 8191), heads, kv_heads, dim, rot, cache, act, rng.random() < 0.4, page, rng.random() < 0.4)
    elif op == "attend":
        new = rng.choice([1, 1, 1, _log(rng, 2, 16)])
        # no more keys in all than the largest listed case has for its heads and rows
        keys = int(5e8 / (kv_heads * dim + 8 * heads * new))
        hi = _log(rng, 1, min(131072, keys))
        seqs = _log(rng, 1, max(1, min(128, keys // hi)))
        c = _attend("", seqs, new, rng.choice([hi, rng.randint(0, hi)]), hi, heads, kv_heads, dim, cache, act, page,
                    new > 1 and rng.random() < 0.5)
    else:
        mixed = rng.random() < 0.4
        c = _sample("", _log(rng, 1, 64), _log(rng, 1000, 248320), 0.0 if mixed else round(rng.uniform(0.3, 1.5), 3),
                    rng.choice([0, 1, _log(rng, 2, 1000)]), rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                    rng.choice([0.0, round(rng.uniform(0.01, 0.3), 3)]), rng.choice([0, 0, rng.randint(1, 31)]))
    del c["name"]
    return c


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _normal(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device=_DEV) * scale).to(dtype)


def _cached(g, case, *shape):
    """Random values as a cache holds them: about unit size, quantized by the scale for 8 bits."""
    kind = _CACHE[case["cache"]][0]
    if kind == torch.float8_e4m3fn:
        out = torch.empty(shape, dtype=torch.uint8, device=_DEV)
        flat = out.view(-1)
        step = 1 << 26
        for at in range(0, flat.numel(), step):   # in pieces: the fp32 source of a large pool need not exist at once
            n = min(step, flat.numel() - at)
            flat[at:at + n] = (_normal(g, n) * 16.0).clamp(-448, 448).to(kind).view(torch.uint8)
        return out.view(kind)
    return torch.randn(*shape, generator=g, device=_DEV, dtype=kind)


def _scales(case):
    return (1.0 / 16.0, 1.0 / 16.0) if case["cache"] == "e4m3" else (1.0, 1.0)


def prepare(case, seed):
    g = torch.Generator(device=_DEV).manual_seed(int(seed))
    s = dict(case)
    act = torch.float32 if case.get("act", "f32") == "f32" else torch.bfloat16
    if case["op"] == "append":
        n, heads, kvh, dim, page = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["page"]
        wide = 2 if case["gated"] else 1
        s["q"] = _normal(g, n, heads, wide, dim, scale=1.5, dtype=act)    # [.., 0, :] are the queries, [.., 1, :] their gates
        s["k"], s["v"] = _normal(g, n, kvh, dim, scale=1.5, dtype=act), _normal(g, n, kvh, dim, dtype=act)
        s["qw"], s["kw"] = 1.0 + 0.1 * _normal(g, dim), 1.0 + 0.1 * _normal(g, dim)
        pairs = case["rot"] // 2
        s["freqs"] = 1e7 ** (-torch.arange(pairs, device=_DEV, dtype=torch.float64) / pairs)
        first = int(torch.randint(0, 200000, (1,), generator=g, device=_DEV))
        s["pos"] = (first + torch.arange(n, device=_DEV)).to(torch.int32)
        pages = (n + page - 1) // page + 2
        order = torch.randperm(pages, generator=g, device=_DEV)
        at = torch.arange(n, device=_DEV) + page // 2                     # the chunk begins inside a page
        s["slots"] = order[at // page] * page + at % page
        kind = _CACHE[case["cache"]][0]
        s["kc"] = torch.zeros(pages, kvh, page, dim, device=_DEV, dtype=torch.uint8 if kind.itemsize == 1 else kind).view(kind)
        s["vc"] = s["kc"].clone()
        s["q_out"] = torch.empty(n, heads, dim, device=_DEV, dtype=act)
    elif case["op"] == "attend":
        n, kvh, dim, page = case["seqs"], case["kv_heads"], case["dim"], case["page"]
        lens = torch.randint(case["kv_lo"], case["kv_hi"] + 1, (n,), generator=g, device=_DEV)
        lens[0] = case["kv_hi"]
        if n > 1:
            lens[-1] = case["kv_lo"]
        s["kv_lens"] = lens.to(torch.int32)
        per = torch.full((n,), case["new"], device=_DEV)
        if case["ragged"]:                                                # the first has all its drafts, others fewer
            per = case["new"] - torch.arange(n, device=_DEV) * 5 % case["new"]
        s["starts"] = torch.cat([torch.zeros(1, device=_DEV, dtype=torch.int64), per.cumsum(0)]).to(torch.int32)
        s["rows"] = int(s["starts"][-1])
        s["wide"] = (case["kv_hi"] + page - 1) // page
        need = (lens + page - 1) // page                                  # a sequence's pages lie anywhere in the pool
        pages = int(need.sum()) + 1
        order = torch.randperm(pages, generator=g, device=_DEV)
        before = need.cumsum(0) - need
        col = torch.arange(s["wide"], device=_DEV)
        s["table"] = torch.where(col < need[:, None], order[(before[:, None] + col).clamp(max=pages - 1)], 0).to(torch.int32)
        s["kc"], s["vc"] = _cached(g, case, pages, kvh, page, dim), _cached(g, case, pages, kvh, page, dim)
        s["q"] = _normal(g, s["rows"], case["heads"], dim, scale=2.0, dtype=act)
        s["out"] = torch.empty(s["rows"], case["heads"], dim, device=_DEV, dtype=act)
    else:
        b, vocab = case["batch"], case["vocab"]
        z = _normal(g, b, vocab + case["pad"], scale=2.0)
        # a few dozen likely tokens above the bulk, as a language model's logits have them
        top = torch.randint(0, vocab, (b, 48), generator=g, device=_DEV)
        z.scatter_(1, top, 12.0 + 2.5 * _normal(g, b, 48))
        s["logits"] = z[:, :vocab]
        full = lambda v, t: torch.full((b,), v, device=_DEV, dtype=t)  # noqa: E731
        s["u"] = torch.rand(b, generator=g, device=_DEV)
        if case["temp"] == 0.0:   # mixed: every row has its own settings, every fifth is greedy
            r = torch.arange(b, device=_DEV)
            pick = lambda vals, t: torch.tensor(vals, device=_DEV, dtype=t)[torch.randint(0, len(vals), (b,), generator=g, device=_DEV)]  # noqa: E731
            s["temp"] = torch.where(r % 5 == 4, torch.zeros((), device=_DEV), pick([0.5, 0.7, 1.0, 1.3], torch.float32))
            s["top_k"], s["top_p"] = pick([0, 1, 20, 50, 400], torch.int32), pick([0.5, 0.8, 0.95, 1.0], torch.float32)
            s["min_p"] = pick([0.0, 0.0, 0.05, 0.2], torch.float32)
        else:
            s["temp"], s["top_k"] = full(case["temp"], torch.float32), full(case["top_k"], torch.int32)
            s["top_p"], s["min_p"] = full(case["top_p"], torch.float32), full(case["min_p"], torch.float32)
        s["pairs"] = torch.zeros(b, 2, device=_DEV, dtype=torch.int32)
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------

def _plain_head(x, w, s):
    """RMS norm of the last axis, then the rotation of its first `rot` elements."""
    x = x.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w
    angle = s["pos"].double()[:, None, None] * s["freqs"]                 # [tokens, 1, pairs]; 64 bits: positions are far
    cos, sin = angle.cos().float(), angle.sin().float()
    rot, half = s["rot"], s["rot"] // 2
    if s["interleaved"]:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, y[..., rot:]], -1)


def _to_cache(x, scale, kind):
    if kind == torch.float8_e4m3fn:
        return (x / scale).clamp(-448, 448).to(kind).view(torch.uint8)
    return x.to(kind)


def _plain_append(s):
    kind = _CACHE[s["cache"]][0]
    ks, vs = _scales(s)
    q = _plain_head(s["q"][:, :, 0], s["qw"], s).to(s["q"].dtype)
    k = _to_cache(_plain_head(s["k"], s["kw"], s), ks, kind)
    v = _to_cache(s["v"].float(), vs, kind)
    page, at = s["slots"] // s["page"], s["slots"] % s["page"]
    raw = torch.uint8 if kind.itemsize == 1 else kind
    s["kc"].view(raw)[page, :, at] = k
    s["vc"].view(raw)[page, :, at] = v
    return {"q": q, "k_cache": s["kc"], "v_cache": s["vc"]}


def _plain_attend(s):
    n, new, kvh, dim, heads = s["seqs"], s["new"], s["kv_heads"], s["dim"], s["heads"]
    group, rows = heads // kvh, s["new"] * (heads // kvh)
    ks, vs = _scales(s)
    starts, lens = s["starts"].long(), s["kv_lens"].long()
    count = starts[1:] - starts[:-1]
    off = torch.arange(new, device=_DEV)
    src = (starts[:-1, None] + off).clamp(max=s["rows"] - 1)              # [seqs, new] rows of q, those behind a sequence's own unused
    q = s["q"].float()[src].view(n, new, kvh, group, dim).permute(0, 2, 1, 3, 4).reshape(n, kvh, rows, dim)
    raw = torch.uint8 if s["kc"].dtype.itemsize == 1 else s["kc"].dtype
    gather = lambda c: c.view(raw)[s["table"].long()].view(c.dtype).float().transpose(1, 2).reshape(n, kvh, -1, dim)  # noqa: E731
    k = gather(s["kc"]) * ks
    score = torch.matmul(k, q.transpose(2, 3).contiguous()) * dim ** -0.5  # [seqs, kv_heads, keys, rows]
    del k
    key = torch.arange(score.shape[2], device=_DEV)
    last = lens[:, None] - count[:, None] + off                           # [seqs, new]: the last key a row sees
    seen = (key[None, :, None] <= last[:, None, :]) & (key[None, :, None] < lens[:, None, None])
    seen = seen.repeat_interleave(group, 2)[:, None]
    score = score.masked_fill(~seen, float("-inf"))
    top = score.amax(2, keepdim=True)
    p = torch.exp(score - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    del score
    total = p.sum(2)                                                       # [seqs, kv_heads, rows]
    v = gather(s["vc"]) * vs
    o = torch.matmul(p.transpose(2, 3).contiguous(), v)
    o = torch.where(total[..., None] > 0, o / total[..., None].clamp(min=1e-30), torch.zeros_like(o))
    o = o.view(n, kvh, new, group, dim).permute(0, 2, 1, 3, 4).reshape(n, new, heads, dim)
    return {"out": o[off < count[:, None]].to(s["q"].dtype)}


def _plain_sample(s):
    z = s["logits"].double()                                               # 64 bits: long sums, and values next to a border
    greedy = ~(s["temp"] > 0)
    t = torch.where(greedy, torch.ones_like(s["temp"]), s["temp"]).double()[:, None]
    ranked, order = torch.sort(z, dim=1, descending=True, stable=True)
    p = torch.exp((ranked - ranked[:, :1]) / t)
    rank = torch.arange(z.shape[1], device=_DEV)[None]
    k = torch.where(s["top_k"] > 0, s["top_k"], z.shape[1])[:, None]
    kept = rank < k
    mass = torch.where(kept, p, 0.0)
    run_sum = mass.cumsum(1)
    top_p = s["top_p"].double()[:, None]
    kept &= (top_p >= 1) | (run_sum - mass < top_p * run_sum[:, -1:]) | (rank == 0)
    kept &= p >= s["min_p"].double()[:, None].clamp(max=1.0)
    kept = torch.where(greedy[:, None], rank == 0, kept)
    weight = torch.zeros_like(p).scatter_(1, order, torch.where(kept, p, 0.0))
    below = weight.cumsum(1)
    token = (below <= s["u"].double()[:, None] * below[:, -1:]).sum(1).clamp(max=z.shape[1] - 1)
    return {"token": token.to(torch.int32), "logit": s["logits"].gather(1, token[:, None])[:, 0]}


# ---- the library's calls --------------------------------------------------------------------------------------------

def _library():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kvmem-qw3_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import q8mi
    return q8mi


def _cache_descriptor(q8mi, s):
    """What a program keeps of a layer's cache."""
    ks, vs = _scales(s)
    pages, kvh, page, dim = s["kc"].shape
    return q8mi.KvCache(k=s["kc"].data_ptr(), v=s["vc"].data_ptr(), dtype=_CACHE[s["cache"]][1], pages=pages, page_size=page,
                        kv_heads=kvh, head_dim=dim, stride_page=kvh * page * dim, stride_head=page * dim, stride_token=dim,
                        k_scale=ks, v_scale=vs)


def _plan(s):
    """The handles that a program sets up once: the library, the cache's descriptor and the workspace."""
    q8mi = _library()
    plan = {"q8mi": q8mi, "lib": q8mi.lib()}
    if s["op"] in ("append", "attend"):
        plan["cache"] = C.byref(_cache_descriptor(q8mi, s))
    if s["op"] == "attend":
        n = plan["lib"].q8mi_paged_attention_scratch_bytes(s["seqs"], s["new"], s["heads"], s["kv_heads"], s["dim"], max(1, s["kv_hi"]))
    elif s["op"] == "sample":
        n = plan["lib"].q8mi_sample_scratch_bytes(s["batch"], s["vocab"])
    else:
        n = 0
    plan["scratch"] = torch.empty(max(16, n), device=_DEV, dtype=torch.uint8)
    return plan


def _own_append(s, p, stream):
    dim = s["dim"]
    wide = s["q"].shape[2]
    p["q8mi"].ok(p["lib"].q8mi_qk_norm_rope_append(
        s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["q_out"].data_ptr(), int(s["act"] == "bf16"), s["tokens"],
        s["heads"], s["heads"] * wide * dim, wide * dim, s["kv_heads"] * dim, s["kv_heads"] * dim, s["heads"] * dim,
        s["qw"].data_ptr(), s["kw"].data_ptr(), _EPS, s["freqs"].data_ptr(), s["rot"], int(s["interleaved"]),
        s["pos"].data_ptr(), s["slots"].data_ptr(), p["cache"], stream), "qk_norm_rope_append")
    return {"q": s["q_out"], "k_cache": s["kc"], "v_cache": s["vc"]}


def _own_attend(s, p, stream):
    bf16, row = int(s["act"] == "bf16"), s["heads"] * s["dim"]
    p["q8mi"].ok(p["lib"].q8mi_paged_attention(
        s["q"].data_ptr(), bf16, s["rows"], row, p["cache"], s["table"].data_ptr(), s["wide"], s["kv_lens"].data_ptr(),
        s["starts"].data_ptr(), s["seqs"], s["new"], s["heads"], s["kv_hi"], s["dim"] ** -0.5, s["out"].data_ptr(), bf16, row,
        p["scratch"].data_ptr(), stream), "paged_attention")
    return {"out": s["out"]}


def _own_sample(s, p, stream):
    p["q8mi"].ok(p["lib"].q8mi_sample(
        s["logits"].data_ptr(), s["batch"], s["vocab"], s["logits"].stride(0), s["temp"].data_ptr(), s["top_k"].data_ptr(),
        s["top_p"].data_ptr(), s["min_p"].data_ptr(), s["u"].data_ptr(), s["pairs"].data_ptr(), p["scratch"].data_ptr(),
        stream), "sample")
    return {"token": s["pairs"][:, 1], "logit": s["pairs"].view(torch.float32)[:, 0]}


def run(state):
    if own:
        if "plan" not in state:
            state["plan"] = _plan(state)
        call = {"append": _own_append, "attend": _own_attend, "sample": _own_sample}[state["op"]]
        return call(state, state["plan"], torch.cuda.current_stream().cuda_stream)
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[state["op"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def _mean_keys(case):
    """Keys that a case's sequences hold together, in the mean (the first has kv_hi, the last kv_lo)."""
    n, lo, hi = case["seqs"], case["kv_lo"], case["kv_hi"]
    return hi if n == 1 else hi + lo + (n - 2) * (lo + hi) / 2


def work(case):
    size = {"f32": 4, "bf16": 2}[case.get("act", "f32")]
    if case["op"] == "append":
        n, h, kvh, dim = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        held = _CACHE[case["cache"]][0].itemsize
        return {"bytes": n * dim * (2 * h * size + 2 * kvh * size + 2 * kvh * held) + 12 * n, "flops": n * dim * (h + kvh) * 8}
    if case["op"] == "attend":
        held, dim = _CACHE[case["cache"]][0].itemsize, case["dim"]
        new = (1 + case["new"]) / 2 if case["ragged"] else case["new"]
        keys = _mean_keys(case)
        return {"bytes": int(2 * keys * case["kv_heads"] * dim * held + 2 * case["seqs"] * new * case["heads"] * dim * size),
                "flops": int(4 * keys * new * case["heads"] * dim)}
    return {"bytes": case["batch"] * (case["vocab"] * 4 + 28), "flops": case["batch"] * case["vocab"] * 4}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](s)


def _exact_append(s):
    def turned(x, w):
        x = x.double()
        y = x / ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + _EPS).sqrt() * w.double()
        pairs = s["rot"] // 2
        first = torch.arange(pairs, device=_DEV) * (2 if s["interleaved"] else 1)
        second = first + (1 if s["interleaved"] else pairs)
        z = torch.complex(y[..., first], y[..., second])
        z = z * torch.polar(torch.ones((), device=_DEV, dtype=torch.float64), s["pos"].double()[:, None] * s["freqs"])[:, None]
        y[..., first], y[..., second] = z.real, z.imag
        return y

    ks, vs = _scales(s)
    out = {"q": turned(s["q"][:, :, 0], s["qw"])}
    for name, x, scale in (("k_cache", turned(s["k"], s["kw"]), ks), ("v_cache", s["v"].double(), vs)):
        pages, kvh, page, dim = s["kc"].shape
        flat = torch.zeros(pages * page, kvh, dim, device=_DEV, dtype=torch.float64)
        flat[s["slots"]] = x / scale
        out[name] = flat.view(pages, page, kvh, dim).transpose(1, 2).contiguous()
    return out


def _exact_attend(s):
    kvh, dim, heads, page = s["kv_heads"], s["dim"], s["heads"], s["page"]
    ks, vs = _scales(s)
    out = torch.zeros(s["rows"], heads, dim, device=_DEV, dtype=torch.float64)
    starts, lens = s["starts"].tolist(), s["kv_lens"].tolist()
    raw = torch.uint8 if s["kc"].dtype.itemsize == 1 else s["kc"].dtype
    for i in range(s["seqs"]):
        n, count = lens[i], starts[i + 1] - starts[i]
        ids = s["table"][i, :(n + page - 1) // page].long()
        for h in range(kvh):
            take = lambda c: c.view(raw)[ids, h].view(c.dtype).reshape(-1, dim)[:n].to(torch.float64)  # noqa: E731
            if n == 0:
                continue
            k, v = take(s["kc"]) * ks, take(s["vc"]) * vs
            for r in range(count):
                see = n - count + r + 1
                if see <= 0:
                    continue
                lo, hi = h * (heads // kvh), (h + 1) * (heads // kvh)
                w = torch.softmax(s["q"][starts[i] + r, lo:hi].double() @ k[:see].T.contiguous() / dim ** 0.5, -1)
                out[starts[i] + r, lo:hi] = w @ v[:see]
    return {"out": out}


def _exact_sample(s):
    tokens = []
    for r in range(s["batch"]):
        z = s["logits"][r].double().cpu()
        temp, u = float(s["temp"][r]), float(s["u"][r])
        order = torch.argsort(-z, stable=True)
        if temp <= 0:
            tokens.append(int(order[0]))
            continue
        p = ((z[order] - z[order[0]]) / temp).exp()
        kept = z.numel()
        if int(s["top_k"][r]) > 0:
            kept = min(kept, int(s["top_k"][r]))
        top_p, min_p = float(s["top_p"][r]), min(1.0, float(s["min_p"][r]))
        if top_p < 1:
            upto = p[:kept].cumsum(0)
            kept = min(kept, 1 + int((upto < top_p * upto[-1]).sum()))
        kept = min(kept, int((p >= min_p).sum()))
        ids, back = torch.sort(order[:kept])
        mass = p[:kept][back].cumsum(0)
        tokens.append(int(ids[min(kept - 1, int(torch.searchsorted(mass, u * mass[-1], right=True)))]))
    token = torch.tensor(tokens, device=_DEV, dtype=torch.int32)
    return {"token": token, "logit": s["logits"].gather(1, token.long()[:, None])[:, 0].double()}
