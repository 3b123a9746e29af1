"""Windowed attention and the microscaled KV cache: what is measured.

Three operators, each one call that a serving program makes per layer:

* ``window`` -- ``run(q, layer, window_left=, sink_tokens=)`` of a planned wrapper: a query at position i sees the
  keys in [i - window_left, i] and the first ``sink_tokens`` of its request; without ``causal`` also those behind it;
* ``store``  -- ``set_kv_cache`` of new tokens into a cache of 8- or 4-bit codes with a shared power-of-two scale
  for every 32 elements, then ``read_kv_cache`` of the requests' whole contexts;
* ``attend`` -- ``run`` over such a cache, with or without a window.

A case gives the batch: ``chunks`` requests of ``new`` tokens over ``prefix`` cached ones, then ``decodes`` one-token
requests of ``ctx`` tokens, lengths drawn by ``lens``.  ``window`` counts the visible keys up to the query's own (0: all).
"""

import math

import numpy as np
import torch

own = False

WORKSPACE_BYTES = 512 << 20
TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "fp8": torch.float8_e4m3fn}
BITS = {"bf16": 16, "f16": 16, "fp8": 8, "mx8": 8.25, "mx4": 4.25}  # of one cached element, its share of a scale included
BLOCK = 32  # elements that share a scale
# largest magnitude that still rounds to a code, exponent of the smallest normal, mantissa bits, largest code
FORMATS = {"mx8": (464.0, -6, 3, 448.0), "mx4": (7.0, 0, 1, 6.0)}


def _case(name, op, heads, kv, *, q="bf16", page=16, window=0, sinks=0, causal=True, chunks=0, new=(0, 0),
          prefix=(0, 0), decodes=0, ctx=(0, 0), lens=0):
    case = {"op": op, "q_heads": heads[0], "kv_heads": heads[1], "head_dim": heads[2], "kv": kv, "q": q, "page": page,
            "window": window, "sinks": sinks, "causal": causal, "chunks": chunks, "new_lo": new[0], "new_hi": new[1],
            "prefix_lo": prefix[0], "prefix_hi": prefix[1], "decodes": decodes, "ctx_lo": ctx[0], "ctx_hi": ctx[1],
            "lens": lens}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one user far into a conversation: the window's few keys, so launches and latency are all there is
        _case("window_decode_b1", "window", (32, 4, 128), "bf16", window=1024, sinks=4, decodes=1, ctx=(32768, 32768)),
        # Orpheus (Llama-3.2-3B) shaped streams at a middling batch, some shorter than their window
        _case("window_decode_b64", "window", (24, 8, 128), "bf16", window=1024, sinks=4, decodes=64, ctx=(128, 4096),
              lens=1),
        # Qwen3-Omni thinker shaped serving at full batch behind a long window
        _case("window_decode_b256", "window", (32, 4, 128), "bf16", window=8192, sinks=64, decodes=256,
              ctx=(512, 32768), lens=2),
        # BAGEL (Qwen2.5-7B) shaped continuous batching: prefill chunks among decode requests
        _case("window_mixed", "window", (28, 4, 128), "bf16", window=2048, sinks=16, chunks=8, new=(512, 2048),
              prefix=(0, 8192), decodes=120, ctx=(1024, 16384), lens=3),
        # long prompts at head_dim 256, in local layers without sinks
        _case("window_chunks_d256", "window", (16, 2, 256), "bf16", window=1024, chunks=8, new=(2048, 2048),
              prefix=(2048, 5632), lens=6),
        # the chunk of one arriving request, written and its context handed on
        _case("store_mx8_chunk", "store", (24, 8, 128), "mx8", chunks=1, new=(500, 500), prefix=(1500, 1500)),
        # chunks of a full batch over long prefixes in 4 bits
        _case("store_mx4_b8", "store", (32, 4, 128), "mx4", chunks=8, new=(512, 2048), prefix=(2048, 16384), lens=5),
        # a handful of short chats in 4 bits
        _case("attend_mx4_b8", "attend", (8, 2, 128), "mx4", decodes=8, ctx=(16, 512)),
        # Orpheus shaped decode over 8 bits
        _case("attend_mx8_b64", "attend", (24, 8, 128), "mx8", decodes=64, ctx=(128, 4096), lens=1),
        # Qwen3-Omni thinker shaped decode at full batch, four times the context in the same memory
        _case("attend_mx4_b256", "attend", (32, 4, 128), "mx4", decodes=256, ctx=(1024, 32768), lens=4),
        # prefill chunks over 8 bits
        _case("attend_mx8_chunks", "attend", (32, 4, 128), "mx8", chunks=4, new=(512, 2048), prefix=(0, 8192), lens=5),
        # a window over 4 bits at head_dim 256: what a long stream on a small share of the memory does
        _case("attend_mx4_window", "attend", (16, 2, 256), "mx4", window=4096, sinks=4, decodes=96, ctx=(2048, 32768),
              lens=7),
    ]


HEADS = [(8, 2, 128), (24, 8, 128), (32, 4, 128), (28, 4, 128), (8, 1, 256), (16, 2, 256), (16, 4, 64)]
MOST_BYTES, MOST_FLOPS = 2.5e9, 3e11


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["window_decode", "window_chunks", "window_mixed", "store", "attend_decode", "attend_chunks",
                       "attend_window"])
    op, mx = kind.split("_")[0], rng.choice(["mx8", "mx4"])
    while True:
        heads, page, lens = rng.choice(HEADS), rng.choice([16, 16, 16, 32, 64, 128]), rng.randrange(1 << 20)
        kw = {"page": page, "lens": lens}
        kv = rng.choice(["bf16", "bf16", "f16", "fp8"]) if op == "window" else mx
        kw["q"] = kv if kv in ("bf16", "f16") else rng.choice(["bf16", "bf16", "f16"])
        if op == "window" or kind == "attend_window":
            kw["window"], kw["sinks"] = _log(rng, 1, 8192), rng.choice([0, 1, 4, _log(rng, 1, 256)])
        if kind in ("window_decode", "attend_decode", "attend_window"):
            hi = _log(rng, 64, 32768)
            kw.update(decodes=_log(rng, 1, 256), ctx=(max(1, hi // _log(rng, 1, 64)), hi))
        else:
            lo = _log(rng, 1, 1024)
            kw.update(chunks=_log(rng, 1, 8), new=(lo, max(lo, _log(rng, 32, 2048))), prefix=(0, _log(rng, 16, 8192)))
            if kind == "window_mixed":
                hi = _log(rng, 256, 16384)
                kw.update(decodes=_log(rng, 1, 120), ctx=(hi // _log(rng, 2, 32), hi))
            elif op != "store":
                kw["causal"] = rng.random() < 0.75
        c = _case(None, op, heads, kv, **kw)
        w = work(c)
        kv_len = _lengths(c)[0]
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS and int(kv_len.sum()) * heads[1] * heads[2] <= 1.2e9:
            return c


def _lengths(case):
    """(tokens after the append, new tokens) of each request."""
    r = np.random.default_rng(case["lens"])

    def between(lo, hi, n):
        return np.rint(np.exp(r.uniform(math.log(max(lo, 1)), math.log(max(hi, 1)), n))).astype(np.int64)

    new = between(case["new_lo"], case["new_hi"], case["chunks"])
    prefix = r.integers(case["prefix_lo"], case["prefix_hi"] + 1, case["chunks"])
    one = np.ones(case["decodes"], np.int64)
    return (np.concatenate([prefix + new, between(case["ctx_lo"], case["ctx_hi"], case["decodes"])]),
            np.concatenate([new, one]))


def work(case):
    kv_len, new = _lengths(case)
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    row = 2 * hkv * d * BITS[case["kv"]] / 8  # K and V of one cached token
    if case["op"] == "store":
        total, n = int(kv_len.sum()), int(new.sum())
        # new rows in and into the cache, the prefixes' codes in, every context out
        return {"bytes": int(n * hkv * d * 4 + total * row + total * hkv * d * 4), "flops": 0}
    window, sinks = case["window"] or 1 << 40, case["sinks"] if case["window"] else 0
    keys = pairs = 0
    for length, n in zip(kv_len.tolist(), new.tolist()):
        at = np.arange(length - n, length)
        first = np.maximum(0, at - window + 1)
        pairs += int(((at + 1 if case["causal"] else length) - first + np.minimum(first, sinks)).sum())
        keys += int(length - first[0] + min(first[0], sinks))
    return {"bytes": int(keys * row + 2 * int(new.sum()) * hq * d * 2), "flops": 4 * d * hq * pairs}


# ------------------------------------------------------------------ inputs
def _codes(x, kind):
    """(codes, scales) of x [..., head_dim] in 32 bits: the plain form of what the cache is written with."""
    most, low, mantissa, top = FORMATS[kind]
    b = x.float().unflatten(-1, (-1, BLOCK))
    m, e = torch.frexp(b.abs().amax(-1))
    tm, te = math.frexp(most)
    e = torch.where(m <= tm, e - te, e - te + 1).clamp(-126, 127)  # the smallest at which the largest still rounds to a code
    y = torch.ldexp(b, -e.unsqueeze(-1)).clamp(-top, top).flatten(-2)
    if kind == "mx8":
        codes = y.to(torch.float8_e4m3fn).view(torch.uint8)
    else:  # 0 0.5 1 1.5 2 3 4 6 by the midpoints between them; a tie goes to the even code
        a = y.abs()
        c = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)).to(torch.uint8)
        c = c | (torch.signbit(y).to(torch.uint8) << 3)
        codes = c[..., 0::2] | (c[..., 1::2] << 4)
    scales = torch.where(b.abs().amax(-1) == 0, 127, e + 127).to(torch.uint8)
    return codes, scales


def _values(codes, scales, kind):
    """What codes [..., head_dim] and scales [..., head_dim / 32] stand for, in 32 bits."""
    if kind == "mx8":
        x = codes.view(torch.float8_e4m3fn).float()
    else:
        grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
        x = torch.stack([grid[(codes & 15).int()], grid[(codes >> 4).int()]], -1).flatten(-2)
    return torch.ldexp(x.unflatten(-1, (-1, BLOCK)), scales.int().unsqueeze(-1) - 127).flatten(-2)


def _inputs(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    hkv, d, ps, kind = case["kv_heads"], case["head_dim"], case["page"], case["kv"]
    kv_len, new = _lengths(case)
    pages = -(-kv_len // ps)
    pool = int(pages.sum()) + max(8, int(pages.sum()) // 8)  # the rest of the pool is free or other requests'
    indices = np.random.default_rng(seed).permutation(pool)[: int(pages.sum())].astype(np.int32)
    indptr = np.concatenate([[0], np.cumsum(pages)]).astype(np.int32)
    qo = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    x = {"kv_len": kv_len.tolist(), "new": new.tolist(), "qo": torch.from_numpy(qo), "indptr": torch.from_numpy(indptr),
         "indices": torch.from_numpy(indices), "last": torch.from_numpy((kv_len - (pages - 1) * ps).astype(np.int32)),
         "pages": [torch.from_numpy(indices[a:b].astype(np.int64)).to(dev) for a, b in zip(indptr[:-1], indptr[1:])],
         "k_scale": None, "v_scale": None, "scales": None}
    step = max(1, (1 << 26) // (2 * ps * hkv * d))  # pages made at a time
    if kind in FORMATS:
        x["kv"] = torch.empty(pool, 2, ps, hkv, d if kind == "mx8" else d // 2, dtype=torch.uint8, device=dev)
        x["scales"] = torch.empty(pool, 2, hkv, d // BLOCK, ps, dtype=torch.uint8, device=dev)
    else:
        x["kv"] = torch.empty(pool, 2, ps, hkv, d, dtype=TORCH[kind], device=dev)
    if kind == "fp8":
        x["k_scale"], x["v_scale"] = (4.5 + torch.rand(2, hkv, device=dev, generator=g)) / 448
    for p in range(0, pool, step):
        n = min(step, pool - p)
        part = torch.empty(n, 2, ps, hkv, d, device=dev).normal_(generator=g)
        if kind in FORMATS:
            x["kv"][p:p + n], s = _codes(part, kind)
            x["scales"][p:p + n] = s.permute(0, 1, 3, 4, 2)
        elif kind == "fp8":
            s = torch.stack([x["k_scale"], x["v_scale"]]).view(1, 2, 1, hkv, 1)
            x["kv"][p:p + n] = (part / s).clamp(-448, 448).to(torch.float8_e4m3fn)
        else:
            x["kv"][p:p + n] = part
    n = int(qo[-1])
    x["q"], x["k"], x["v"] = (torch.empty(n, h, d, dtype=TORCH[case["q"]], device=dev).normal_(generator=g)
                              for h in (case["q_heads"], hkv, hkv))
    return x


def prepare(case, seed):
    x = _inputs(case, seed)
    s = {"case": case, "x": x}
    if own:
        from mstar_amd.paged_attention import PagedDecodeWrapper, PagedPrefillWrapper

        dev = x["q"].device
        ws = torch.empty(WORKSPACE_BYTES, dtype=torch.uint8, device=dev)
        heads = (case["q_heads"], case["kv_heads"], case["head_dim"], case["page"])
        if case["chunks"] == 0:
            s["w"] = PagedDecodeWrapper(ws, *heads, device=dev)
            s["w"].plan(x["indptr"], x["indices"], x["last"], dtype=x["q"].dtype)
        else:
            s["w"] = PagedPrefillWrapper(ws, *heads, device=dev)
            s["w"].plan(x["qo"], x["indptr"], x["indices"], x["last"], causal=case["causal"], dtype=x["q"].dtype)
        s["layer"] = x["kv"]
        if case["kv"] in FORMATS:
            from mstar_amd.mx_cache import MXKVLayer

            s["layer"] = MXKVLayer(x["kv"], x["scales"])
        if case["op"] == "store":
            s["on_gpu"] = [x[k].to(dev) for k in ("indptr", "indices", "last")]
    return s


# --------------------------------------------------------------- one pass
def run(s):
    case, x = s["case"], s["x"]
    if own:
        return _own(s, case, x)
    return _plain_store(case, x) if case["op"] == "store" else _plain_attention(case, x)


def _own(s, case, x):
    w, layer = s["w"], s["layer"]
    if case["op"] == "store":
        from mstar_amd.mx_cache import read_kv_cache

        w.set_kv_cache(layer, x["k"], x["v"])
        k, v = read_kv_cache(layer, *s["on_gpu"], sum(x["kv_len"]), dtype=x["q"].dtype)
        return {"k": k, "v": v}
    if case["window"]:
        return w.run(x["q"], layer, x["k_scale"], x["v_scale"], window_left=case["window"] - 1,
                     sink_tokens=case["sinks"])
    return w.run(x["q"], layer)


def _gather(case, x, i, which, at=None):
    """Request i's cached K (which 0) or V (1) at the given positions (all), [tokens, kv_heads, head_dim] in 32 bits."""
    pages = x["pages"][i]
    if at is None:
        at = torch.arange(x["kv_len"][i], device=pages.device)
    page, slot = pages[at // case["page"]], at % case["page"]
    rows = x["kv"][page, which, slot]
    if case["kv"] in FORMATS:
        return _values(rows, x["scales"][page, which, :, :, slot], case["kv"])
    if case["kv"] == "fp8":
        return rows.float() * x["k_scale" if which == 0 else "v_scale"][:, None]
    return rows.float()


def _plain_store(case, x):
    dev, kind, k, v = x["q"].device, case["kv"], [], []
    for i, (length, n) in enumerate(zip(x["kv_len"], x["new"])):
        rows = slice(int(x["qo"][i]), int(x["qo"][i]) + n)
        at = torch.arange(length - n, length, device=dev)
        page, slot = x["pages"][i][at // case["page"]], at % case["page"]
        for which, src in enumerate((x["k"], x["v"])):
            codes, scales = _codes(src[rows], kind)
            x["kv"][page, which, slot] = codes
            x["scales"][page, which, :, :, slot] = scales
        k.append(_gather(case, x, i, 0).to(x["q"].dtype))
        v.append(_gather(case, x, i, 1).to(x["q"].dtype))
    return {"k": torch.cat(k), "v": torch.cat(v)}


def _plain_attention(case, x):
    dev, (hq, hkv, d) = x["q"].device, (case["q_heads"], case["kv_heads"], case["head_dim"])
    window, sinks = case["window"] or 1 << 40, case["sinks"] if case["window"] else 0
    out = torch.empty_like(x["q"])
    for i, (length, n) in enumerate(zip(x["kv_len"], x["new"])):
        rows = slice(int(x["qo"][i]), int(x["qo"][i]) + n)
        first = max(0, length - n - window + 1)
        keys = torch.cat([torch.arange(min(sinks, first), device=dev), torch.arange(first, length, device=dev)])
        at = torch.arange(length - n, length, device=dev)[:, None]
        seen = (keys > at - window) | (keys < sinks)
        if case["causal"] or case["chunks"] == 0:
            seen &= keys <= at
        k, v = (_gather(case, x, i, which, keys).transpose(0, 1) for which in (0, 1))
        q = x["q"][rows].float().view(n, hkv, hq // hkv, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)
        p = torch.matmul(q, k.transpose(1, 2).contiguous()).view(hkv, hq // hkv, n, -1) / math.sqrt(d)
        p = p.masked_fill(~seen, -math.inf)
        p = torch.exp(p - p.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        o = torch.matmul(p.view(hkv, -1, keys.numel()), v).view(hkv, hq // hkv, n, d)
        out[rows] = o.permute(2, 0, 1, 3).reshape(n, hq, d).to(out.dtype)
    return out


# ------------------------------------------------------------------- exact
def _exact_rounded(x, kind):
    """x [tokens, heads, head_dim] in 64 bits, rounded block by block to what the cache holds."""
    most, low, mantissa, top = FORMATS[kind]
    b = x.double().reshape(*x.shape[:-1], -1, BLOCK)
    peak = b.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(peak.clamp_min(2.0 ** -140))) - math.ceil(math.log2(most))
    while True:  # the smallest exponent with peak <= most * 2^e
        more = peak > most * torch.exp2(e)
        if not more.any():
            break
        e = e + more
    scale = torch.exp2(e.clamp(-126, 127))
    y = (b / scale).clamp(-top, top)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** low))) - mantissa)
    return (torch.round(y / step) * step * scale).reshape(x.shape)


def _exact_values(case, x, rows, scales, which):
    if case["kv"] == "mx8":
        rows = rows.view(torch.float8_e4m3fn).double()
    elif case["kv"] == "mx4":
        both = torch.stack([rows & 15, rows >> 4], -1).reshape(*rows.shape[:-1], -1).long()
        mag, low = both & 7, (both & 7) < 2
        value = torch.where(low, mag * 0.5, (1 + (mag & 1) * 0.5) * torch.exp2((mag >> 1).double() - 1))
        rows = torch.where(both > 7, -value, value)
    elif case["kv"] == "fp8":
        return rows.double() * (x["k_scale"], x["v_scale"])[which].double()[None, :, None]
    else:
        return rows.double()
    return rows * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, -1)


def exact(case, seed):
    x = _inputs(case, seed)
    ps, hq, hkv, d = case["page"], case["q_heads"], case["kv_heads"], case["head_dim"]
    out, store = [], {"k": [], "v": []}
    for i, (length, n) in enumerate(zip(x["kv_len"], x["new"])):
        q0 = int(x["qo"][i])
        context = []
        for which in (0, 1):
            rows = x["kv"][x["pages"][i], which].reshape(-1, hkv, x["kv"].shape[-1])[:length]
            scales = None
            if x["scales"] is not None:
                scales = x["scales"][x["pages"][i], which].permute(0, 3, 1, 2).reshape(-1, hkv, d // BLOCK)[:length]
            context.append(_exact_values(case, x, rows, scales, which))
        if case["op"] == "store":
            for which, name in enumerate(("k", "v")):
                context[which][length - n:] = _exact_rounded(x[name][q0:q0 + n], case["kv"])
                store[name].append(context[which])
            continue
        o = torch.empty(n, hq, d, dtype=torch.float64, device=x["q"].device)
        for a in range(0, n, 512):  # rows at a time
            b = min(n, a + 512)
            at = torch.arange(length - n + a, length - n + b, device=o.device).unsqueeze(1)
            key = torch.arange(length, device=o.device).unsqueeze(0)
            hidden = torch.zeros(b - a, length, dtype=torch.bool, device=o.device)
            if case["causal"] or case["chunks"] == 0:
                hidden |= key > at
            if case["window"]:
                hidden |= (at - key >= case["window"]) & (key >= case["sinks"])
            use = (~hidden).any(0).nonzero().squeeze(1)
            for h in range(hkv):
                k, v = (c[use, h] for c in context)
                for j in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                    score = x["q"][q0 + a:q0 + b, j].double() @ k.T * d ** -0.5
                    score[hidden[:, use]] = -math.inf
                    o[a:b, j] = torch.softmax(score, -1) @ v
        out.append(o)
    return {name: torch.cat(parts) for name, parts in store.items()} if case["op"] == "store" else torch.cat(out)
