"""Attention of new tokens over a paged cache, and the cache in 8 bits: cases for timing.

Four operators that work on one paged KV cache: ``paged_prefill`` (a chunk of
new tokens of every sequence attends its pages), ``quantize_and_cache`` (the
write into an 8-bit cache, one scale for each token and kv head),
``gather_cache`` (reading pages back as packed rows) and ``paged_decode_split``
over an 8-bit cache with such scales (single tokens). ``listed()`` names the
cases, ``draw(rng)`` gives others of the same ranges; ``prepare`` makes one
case's inputs, ``run`` is one pass (the plain form in elementary torch
operations, or, where ``own`` is true, the framework's calls), ``exact`` the
outputs' values in 64 bits.
"""

import math
import types

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
TOP = {"fp8": 448.0, "int8": 127.0}  # the largest code
LEAST_SCALE = 2.0 ** -126
# A drawn attention costs at most this many operations, any drawn case at most this many cache
# bytes (the largest listed cases': 2.1e12 and 0.4e9).
MOST_FLOPS = 1.2e12
MOST_BYTES = 0.3e9
# Score elements that the plain form holds at once.
BLOCK = 1 << 28


def _case(name, kind, batch, q_heads, kv_heads, head_dim, dtype, cache, lo, hi, **more):
    """One case. lo, hi: tokens that a sequence holds in the cache before the call (uniform
    integers); new_lo, new_hi: its new tokens (the first ``decodes`` sequences have one); cache:
    "16" (the dtype itself), "fp8" or "int8"; window, softcap, sinks, alibi: attention's options;
    pad: slots of -1 at the end of a write."""
    case = dict(kind=kind, batch=batch, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                dtype=dtype, cache=cache, lo=lo, hi=hi, new_lo=1, new_hi=1, decodes=0,
                page_size=16, window=-1, softcap=0.0, sinks=False, alibi=False, pad=0)
    case.update(more)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # A short follow-up question of one user of a small model: latency.
        _case("chunk_one_short_d64", "prefill", 1, 8, 2, 64, "f16", "16", 83, 83, new_lo=17,
              new_hi=17),
        # Prompts of several users that arrive together, nothing cached before.
        _case("chunk_prompts_d128", "prefill", 6, 32, 8, 128, "bf16", "16", 0, 0, new_lo=300,
              new_hi=1500),
        # One scheduler step of a server with chunked prompts: a chunk of one long prompt beside
        # the single tokens of the requests that decode, over an 8-bit cache.
        _case("chunk_mixed_int8_d128", "prefill", 32, 32, 8, 128, "bf16", "int8", 1024, 8192,
              new_lo=1024, new_hi=1024, decodes=31),
        # A chunk of a long document late in its prompt: the most work.
        _case("chunk_long_d128", "prefill", 1, 32, 8, 128, "bf16", "16", 28672, 28672, new_lo=4096,
              new_hi=4096),
        # A local layer of a model with small heads: sliding window and sinks, ragged chunks.
        _case("chunk_window_d64", "prefill", 3, 32, 4, 64, "f16", "16", 501, 5000, new_lo=700,
              new_hi=2100, window=1023, sinks=True, page_size=64),
        # One layer's two calls for a prompt chunk: its rows written in 8 bits, then attended
        # with those before them.
        _case("layer_chunk_int8_d128", "layer", 2, 32, 8, 128, "bf16", "int8", 1000, 3000,
              new_lo=1024, new_hi=2048),
        # The write of one decode step's tokens, the batch padded for a captured graph.
        _case("write_step_int8_d128", "write", 1, 32, 8, 128, "bf16", "int8", 123, 123, pad=5),
        # The write of a long prompt's rows.
        _case("write_prompt_fp8_d128", "write", 1, 32, 8, 128, "bf16", "fp8", 16384, 16384),
        # Reading a short request's pages back.
        _case("gather_one_fp8_d64", "gather", 1, 16, 8, 64, "f16", "fp8", 777, 777),
        # Reading a batch's whole context back, lengths as they come.
        _case("gather_int8_d128", "gather", 16, 32, 8, 128, "bf16", "int8", 1024, 8192),
        # One request of a small model decoding: latency.
        _case("decode_one_fp8_d64", "decode", 1, 16, 8, 64, "f16", "fp8", 500, 500),
        # The ordinary serving batch on an 8-bit cache.
        _case("decode_int8_d128", "decode", 32, 32, 8, 128, "bf16", "int8", 1024, 8192),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["prefill", "prefill", "prefill", "layer", "write", "gather", "decode",
                       "decode"])
    cache = rng.choice(["fp8", "int8"])
    if kind == "prefill":
        cache = rng.choice(["16", "16", "fp8", "int8"])
    elif kind == "gather":
        cache = rng.choice(["16", "fp8", "int8"])
    head_dim = rng.choice([64, 128, 128, 256] if kind in ("prefill", "decode") else [64, 128])
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    gq = rng.choice([1, 2, 3, 4, 7, 8, 16] if kv_heads < 8 else [1, 2, 4])
    dtype = rng.choice(["f16", "bf16"])
    more = {"page_size": rng.choice([8, 16, 16, 32, 64, 256])}
    row = 2 * kv_heads * head_dim * (2 if cache == "16" else 1)
    if kind in ("write", "gather", "decode"):
        batch = 1 if kind == "write" else _log(rng, 1, 100)
        moved = {"write": 3, "gather": 3, "decode": 1}[kind] * row * batch
        most = max(64, int(min(20000, MOST_BYTES / moved)))
        hi = _log(rng, 1 if kind == "write" else 33, most)
        lo = hi if kind == "write" else rng.choice([1, max(1, hi // 8), hi])
        if kind == "write" and rng.random() < 0.3:
            more["pad"] = rng.randint(1, 9)
    else:
        batch = _log(rng, 1, 24)
        new_hi = _log(rng, 2, 4096)
        more["new_lo"] = rng.choice([1, max(1, new_hi // 3), new_hi])
        more["decodes"] = rng.choice([0, 0, batch // 2]) if kind == "prefill" else 0
        per = batch * new_hi * 4 * kv_heads * gq * head_dim  # operations for each key
        most = min(MOST_FLOPS / per, MOST_BYTES / (row * batch)) - new_hi / 2
        while most < 0:
            new_hi = new_hi // 2 + 1
            batch = (batch + 1) // 2
            more["new_lo"] = min(more["new_lo"], new_hi)
            more["decodes"] = min(more["decodes"], batch // 2)
            per = batch * new_hi * 4 * kv_heads * gq * head_dim
            most = min(MOST_FLOPS / per, MOST_BYTES / (row * batch)) - new_hi / 2
        more["new_hi"] = new_hi
        hi = rng.choice([0, _log(rng, 1, max(1, min(20000, int(most))))])
        lo = rng.choice([0, hi // 4, hi])
        if kind == "prefill":
            if rng.random() < 0.25:
                more["window"] = _log(rng, 16, 4096)
            more["sinks"] = rng.random() < 0.15
            more["alibi"] = rng.random() < 0.1
            more["softcap"] = rng.choice([0.0] * 6 + [30.0])
    return _case(None, kind, batch, kv_heads * gq, kv_heads, head_dim, dtype, cache, lo, hi, **more)


# ---------------------------------------------------------------------------
# Inputs


def _lengths(case):
    """(new tokens, tokens in all) of each sequence: a fixed draw per shape, so that every seed's
    pass does the same work on other values."""
    g = torch.Generator().manual_seed(20261207 + case["batch"])
    b = case["batch"]
    held = torch.randint(case["lo"], case["hi"] + 1, (b,), generator=g)
    new = torch.randint(case["new_lo"], case["new_hi"] + 1, (b,), generator=g)
    new[:case["decodes"]] = 1
    if case["kind"] in ("gather", "decode", "write"):
        return new, held
    return new, held + new


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32)


def _quantise(x, cache):
    """Codes and scales of rows x [..., HD]: scale = max |x| / TOP (at least 2^-126), code =
    x / scale to the nearest, ties to even, all in 32 bits. A row with an infinity or NaN has
    the scale NaN and codes 0."""
    x = x.float()
    # (a tensor divisor: torch multiplies by the reciprocal of a plain number)
    scale = (x.abs().amax(-1) / torch.full((), TOP[cache], device=x.device)).clamp(min=LEAST_SCALE)
    scale = torch.where(scale.isfinite(), scale, torch.full_like(scale, math.nan))
    y = (x / scale[..., None]).clamp(-TOP[cache], TOP[cache]).nan_to_num(0.0)
    return (y.round() if cache == "int8" else y).to(CODES[cache]), scale


def _slots(s, case, first, count, at):
    """Cache slots of the positions first .. first + count - 1 of sequence ``at``."""
    pos = torch.arange(first, first + count, device=DEVICE)
    return s.table[at].to(torch.int64)[pos // case["page_size"]] * case["page_size"] + \
        pos % case["page_size"]


def prepare(case, seed):
    """What the program holds before the call, on the GPU."""
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt, hd, hkv, hq = DTYPES[case["dtype"]], case["head_dim"], case["kv_heads"], case["q_heads"]
    b, ps, kind, cache = case["batch"], case["page_size"], case["kind"], case["cache"]
    new, total = _lengths(case)
    s = types.SimpleNamespace(case=case, kind=kind, new=new.tolist(), lens=total.tolist(),
                              scale=hd ** -0.5)
    # Pages: every sequence's own, from a shuffled pool a quarter larger.
    need = (total + ps - 1) // ps
    pool = math.ceil(1.25 * int(need.sum())) + 1
    perm = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.zeros(b, max(1, int(need.max())), dtype=torch.int32)
    table[torch.arange(table.shape[1])[None, :] < need[:, None]] = perm[:int(need.sum())]
    s.table = table.to(DEVICE)
    s.seqlens = total.to(DEVICE, torch.int32)
    # Keys and values of a layer: rows of different magnitudes, as tokens and heads have them.
    if kind == "write":
        s.kc, s.vc = (torch.zeros(pool, ps, hkv, hd, device=DEVICE, dtype=torch.float32)
                      .to(CODES[cache]) for _ in range(2))
        s.ks, s.vs = (torch.zeros(pool, hkv, ps, device=DEVICE) for _ in range(2))
        n = s.lens[0]
        s.slots = torch.cat([_slots(s, case, 0, n, 0),
                             torch.full((case["pad"],), -1, device=DEVICE)])
        rows = n + case["pad"]
    else:
        sides = []
        for _ in range(2):
            x = _normal(g, pool, ps, hkv, hd)
            if cache == "16":
                sides.append((x.to(dt), None))
                continue
            codes, scale = _quantise(x.mul_(torch.exp(0.5 * _normal(g, pool, ps, hkv, 1))).to(dt),
                                     cache)
            sides.append((codes, scale.permute(0, 2, 1).contiguous()))
        (s.kc, s.ks), (s.vc, s.vs) = sides
        rows = sum(s.new)
    if kind in ("write", "layer"):
        # Slices of one fused projection, as a layer has them.
        kv = (_normal(g, rows, 2 * hkv, hd) *
              torch.exp(0.5 * _normal(g, rows, 2 * hkv, 1))).to(dt)
        s.key, s.value = kv[:, :hkv], kv[:, hkv:]
    if kind == "layer":
        s.slots = torch.cat([_slots(s, case, s.lens[i] - s.new[i], s.new[i], i)
                             for i in range(b)])
    if kind in ("prefill", "layer"):
        s.q = _normal(g, rows, hq, hd).to(dt)
        s.cu = torch.nn.functional.pad(new.cumsum(0), (1, 0)).to(DEVICE, torch.int32)
    if kind == "decode":
        s.q = _normal(g, b, hq, hd).to(dt)
    if kind == "gather":
        s.cu = torch.nn.functional.pad(total.cumsum(0), (1, 0)).to(DEVICE, torch.int32)
    s.sinks = _normal(g, hq) if case["sinks"] else None
    s.alibi = torch.logspace(-1, -8, hq, base=2.0, device=DEVICE) if case["alibi"] else None
    return s


# ---------------------------------------------------------------------------
# The plain form


def _rows(s, i):
    """K and V rows [L, HKV, HD] of sequence i in 32 bits."""
    n, ps = s.lens[i], s.case["page_size"]
    pages = s.table[i, :(n + ps - 1) // ps].to(torch.int64)
    got = []
    for codes, scale in ((s.kc, s.ks), (s.vc, s.vs)):
        x = codes[pages].float()
        if scale is not None:
            x = x * scale[pages].permute(0, 2, 1)[..., None]
        got.append(x.flatten(0, 1)[:n])
    return got


def _attend(s, q, k, v):
    """q [N, HQ, HD]: the last N of the tokens with the keys k, v [L, HKV, HD]; in 32 bits."""
    c = s.case
    n, hq, hd = q.shape
    length, hkv = k.shape[0], k.shape[1]
    gq = hq // hkv
    kt, vt = k.permute(1, 2, 0).contiguous(), v.permute(1, 0, 2).contiguous()
    keys = torch.arange(length, device=DEVICE)
    out = torch.empty(n, hq, hd, device=DEVICE)
    step = max(1, BLOCK // (hq * length))
    for first in range(0, n, step):
        part = q[first:first + step].float()
        m = part.shape[0]
        x = part.view(m, hkv, gq, hd).permute(1, 2, 0, 3).reshape(hkv, gq * m, hd) @ kt * s.scale
        x = x.view(hq, m, length)
        if c["softcap"] > 0:
            x = c["softcap"] * torch.tanh(x / c["softcap"])
        behind = (length - n + first + torch.arange(m, device=DEVICE))[:, None] - keys[None, :]
        if s.alibi is not None:
            x = x - s.alibi[:, None, None] * behind.abs()
        hidden = behind < 0
        if c["window"] >= 0:
            hidden = hidden | (behind > c["window"])
        x = x.masked_fill(hidden, -math.inf)
        top = x.amax(-1, keepdim=True)
        p = torch.exp(x - top)
        total = p.sum(-1, keepdim=True)
        if s.sinks is not None:
            total = total + torch.exp(s.sinks[:, None, None] - top)
        o = (p / total).view(hkv, gq * m, length) @ vt
        out[first:first + m] = o.view(hq, m, hd).permute(1, 0, 2)
    return out


def _write(s):
    keep = s.slots >= 0
    at = s.slots[keep]
    page, off = at // s.case["page_size"], at % s.case["page_size"]
    for x, codes, scale in ((s.key, s.kc, s.ks), (s.value, s.vc, s.vs)):
        c, sc = _quantise(x[keep], s.case["cache"])
        codes.view(torch.uint8)[page, off] = c.view(torch.uint8)
        scale.permute(0, 2, 1)[page, off] = sc


def _decode(s):
    """One query token of each sequence, all sequences padded to the longest."""
    c = s.case
    b, hkv, hd, ps = c["batch"], c["kv_heads"], c["head_dim"], c["page_size"]
    gq = c["q_heads"] // hkv
    at = s.table.to(torch.int64)
    width = at.shape[1] * ps
    hidden = torch.arange(width, device=DEVICE)[None, :] >= s.seqlens[:, None]
    kv = []
    for codes, scale in ((s.kc, s.ks), (s.vc, s.vs)):
        x = codes[at].float() * scale[at].transpose(2, 3)[..., None]
        kv.append(x.reshape(b, width, hkv, hd).transpose(1, 2).reshape(b * hkv, width, hd))
    q = s.q.float().view(b * hkv, gq, hd)
    x = (q @ kv[0].transpose(1, 2) * s.scale).view(b, hkv, gq, width)
    x = x.masked_fill(hidden[:, None, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    return (p.view(b * hkv, gq, width) @ kv[1]).view(b, hkv * gq, hd).to(s.q.dtype)


def _caches(s):
    return {"k_cache": s.kc, "v_cache": s.vc, "k_scale": s.ks, "v_scale": s.vs}


def run(s):
    """One pass of a user's program."""
    if own:
        return _run_own(s)
    if s.kind in ("write", "layer"):
        _write(s)
    if s.kind == "write":
        return _caches(s)
    if s.kind == "decode":
        return _decode(s)
    dt = DTYPES[s.case["dtype"]]
    if s.kind == "gather":
        rows = [_rows(s, i) for i in range(s.case["batch"])]
        return {"k": torch.cat([k for k, _ in rows]).to(dt),
                "v": torch.cat([v for _, v in rows]).to(dt)}
    parts = s.q.split(s.new)
    out = torch.cat([_attend(s, q, *_rows(s, i)) for i, q in enumerate(parts)]).to(dt)
    return {"out": out, **_caches(s)} if s.kind == "layer" else out


def _run_own(s):
    import mxflashattn_amd as mx

    if s.kind in ("write", "layer"):
        mx.quantize_and_cache(s.key, s.value, s.kc, s.vc, s.ks, s.vs, s.slots)
    if s.kind == "write":
        return _caches(s)
    if s.kind == "decode":
        return mx.paged_decode_split(s.q, s.kc, s.vc, s.table, s.seqlens, s.scale, k_scale=s.ks,
                                     v_scale=s.vs)
    if s.kind == "gather":
        k, v = mx.gather_cache(s.kc, s.vc, s.table, s.cu, sum(s.lens), k_scale=s.ks, v_scale=s.vs,
                               dtype=DTYPES[s.case["dtype"]])
        return {"k": k, "v": v}
    c = s.case
    out = mx.paged_prefill(s.q, s.kc, s.vc, s.cu, s.table, s.seqlens, s.scale, causal=True,
                           window_left=c["window"], softcap=c["softcap"], sinks=s.sinks,
                           alibi_slopes=s.alibi, k_scale=s.ks, v_scale=s.vs)
    return {"out": out, **_caches(s)} if s.kind == "layer" else out


def _seen(case):
    """(query-key pairs, keys that some query sees) over all sequences, by arithmetic."""
    pairs = keys = 0
    new, total = _lengths(case)
    for n, length in zip(new.tolist(), total.tolist()):
        w = case["window"]
        first = length - n  # the first query's position: it sees first + 1 keys
        if w < 0:
            pairs += n * first + n * (n + 1) // 2
            keys += length
        else:
            full = min(n, max(0, w - first))  # queries that the window hides nothing from
            pairs += full * first + full * (full + 1) // 2 + (n - full) * (w + 1)
            keys += min(length, w + n)
    return pairs, keys


def work(case):
    hd, hkv, hq, b, kind = (case[k] for k in ("head_dim", "kv_heads", "q_heads", "batch", "kind"))
    wide = case["cache"] == "16"
    row = 2 * hkv * (2 * hd if wide else hd + 4)  # K and V of one token in the cache, with scales
    new, total = _lengths(case)
    if kind == "write":
        return {"bytes": case["hi"] * (4 * hkv * hd + row + 8), "flops": 0}
    if kind == "gather":
        n = int(total.sum())
        pages = int(((total + case["page_size"] - 1) // case["page_size"]).sum())
        return {"bytes": n * (row + 4 * hkv * hd) + 4 * pages + 8 * b, "flops": 0}
    if kind == "decode":
        n = int(total.sum())
        pairs, keys, rows = n, n, b
    else:
        pairs, keys = _seen(case)
        rows = int(new.sum())
    moved = keys * row + 4 * rows * hq * hd + 4 * -(-keys // case["page_size"]) + 8 * b
    if kind == "layer":
        moved += rows * (4 * hkv * hd + row + 8)
    return {"bytes": moved, "flops": 4 * pairs * hq * hd}


# ---------------------------------------------------------------------------
# The same in 64 bits


def _wide_rows(s, i):
    """K and V rows of sequence i as the cache's codes and scales say, in float64."""
    ps = s.case["page_size"]
    pos = torch.arange(s.lens[i], device=DEVICE)
    page, off = s.table[i].long()[pos // ps], pos % ps
    k, v = s.kc[page, off].double(), s.vc[page, off].double()
    if s.ks is not None:
        k, v = k * s.ks[page, :, off].double()[..., None], v * s.vs[page, :, off].double()[..., None]
    return k, v


def _wide_attend(s, q, k, v):
    """Softmax attention of one sequence's last tokens, a query head and some rows at a time."""
    c = s.case
    n, hq, hd = q.shape
    length = k.shape[0]
    gq = hq // k.shape[1]
    out = torch.empty(n, hq, hd, device=DEVICE, dtype=torch.float64)
    key_at = torch.arange(length, device=DEVICE)
    step = max(1, (1 << 27) // length)
    for h in range(hq):
        kh, vh = k[:, h // gq].t().contiguous(), v[:, h // gq].contiguous()
        for a in range(0, n, step):
            e = min(n, a + step)
            x = torch.mm(q[a:e, h].double().contiguous(), kh).mul_(s.scale)
            if c["softcap"] > 0:
                x = torch.tanh(x / c["softcap"]) * c["softcap"]
            at = torch.arange(length - n + a, length - n + e, device=DEVICE)
            far = at[:, None] - key_at[None, :]
            if s.alibi is not None:
                x = x - far.abs() * s.alibi[h].double()
            x.masked_fill_(far < 0, -math.inf)
            if c["window"] >= 0:
                x.masked_fill_(far > c["window"], -math.inf)
            if s.sinks is not None:
                x = torch.cat([x, s.sinks[h].double().expand(e - a, 1)], 1)
            out[a:e, h] = torch.mm(torch.softmax(x, -1)[:, :length].contiguous(), vh)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = s.kind
    scales = {}
    if kind in ("write", "layer"):
        # The scales are numbers of the inputs; a code next to a border goes by 32 bits.
        keep = s.slots >= 0
        page, off = s.slots[keep] // case["page_size"], s.slots[keep] % case["page_size"]
        for name, x, codes, held in (("k", s.key, s.kc, s.ks), ("v", s.value, s.vc, s.vs)):
            top = x[keep].double().abs().amax(-1) / TOP[case["cache"]]
            wide = held.double()
            wide[page, :, off] = top.clamp(min=LEAST_SCALE)
            scales[name + "_scale"] = wide
            scales[name + "_cache"] = None
            if kind == "layer":  # what attention then reads: codes and scales as they are stored
                narrow, sc = _quantise(x[keep], case["cache"])
                codes.view(torch.uint8)[page, off] = narrow.view(torch.uint8)
                held[page, :, off] = sc
    if kind == "write":
        return scales
    if kind == "gather":
        rows = [_wide_rows(s, i) for i in range(case["batch"])]
        return {"k": torch.cat([k for k, _ in rows]), "v": torch.cat([v for _, v in rows])}
    parts = s.q.split(s.new) if kind != "decode" else s.q.split(1)
    out = torch.cat([_wide_attend(s, q, *_wide_rows(s, i)) for i, q in enumerate(parts)])
    return {"out": out, **scales} if kind == "layer" else out
