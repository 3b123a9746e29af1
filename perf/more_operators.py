"""Norm, rotate and store; attention weights of cached tokens; eviction by them: what is measured.

Three operators, each one call that a serving program makes:

* ``norm``    -- ``qk_norm_rope_set_kv_cache`` of a planned wrapper, once a layer: q and k are normalised head by head
  (root mean square, a weight for each element), rotated to their positions, and k and v written to the paged cache;
* ``weights`` -- ``accumulate_weights`` of a planned wrapper, once a layer: the softmax probabilities that the step's
  queries give to every cached token, summed over queries and over the q heads of a kv head, are added to the
  token's weight; the step's own tokens begin at zero;
* ``evict``   -- ``evict_kv_cache`` of all layers, now and then: of each request and kv head the first ``sinks``, the last
  ``recent`` and the heaviest of the tokens between stay, ``keep`` in all, moved to the front in their order.

A case gives the batch: ``chunks`` requests of ``new`` tokens over ``prefix`` cached ones, then ``decodes`` requests of
``ctx`` tokens, the last of them new, lengths drawn by ``lens``.
"""

import math

import numpy as np
import torch

own = False

WORKSPACE_BYTES = 512 << 20
TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "fp8": torch.float8_e4m3fn}
BITS = {"bf16": 16, "f16": 16, "fp8": 8, "mx8": 8.25, "mx4": 4.25}  # of one cached element, its share of a scale included
BLOCK = 32  # elements of a microscaled cache that share a scale
EPS = 1e-6
LLAMA31 = {"low_freq_factor": 1.0, "high_freq_factor": 4.0, "old_context_len": 8192}


def _case(name, op, heads, kv, *, q="bf16", page=16, causal=True, chunks=0, new=(0, 0), prefix=(0, 0), decodes=0,
          ctx=(0, 0), lens=0, rotary=0, interleave=False, llama31=False, theta=1e6, first=0, layers=1, keep=0, recent=0,
          sinks=0):
    case = {"op": op, "q_heads": heads[0], "kv_heads": heads[1], "head_dim": heads[2], "kv": kv, "q": q, "page": page,
            "causal": causal, "chunks": chunks, "new_lo": new[0], "new_hi": new[1], "prefix_lo": prefix[0],
            "prefix_hi": prefix[1], "decodes": decodes, "ctx_lo": ctx[0], "ctx_hi": ctx[1], "lens": lens,
            "rotary": rotary or heads[2], "interleave": interleave, "llama31": llama31, "theta": theta, "first": first,
            "layers": layers, "keep": keep, "recent": recent, "sinks": sinks}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one user's next token, far into a long context: a launch, and what it waits for
        _case("norm_b1", "norm", (32, 4, 128), "bf16", decodes=1, ctx=(16, 16), first=130000),
        # Qwen3-Omni thinker shaped decode at full batch
        _case("norm_b256", "norm", (32, 4, 128), "bf16", decodes=256, ctx=(1, 64), first=30000, lens=1),
        # arriving prompts of odd lengths, half of each head rotated in neighbouring pairs
        _case("norm_chunks_d64", "norm", (16, 4, 64), "f16", q="f16", chunks=5, new=(70, 1500), prefix=(0, 40), rotary=32,
              interleave=True, theta=1e4, lens=2),
        # BAGEL (Qwen2.5-7B with normed heads) shaped prompts, a full step of them
        _case("norm_chunks", "norm", (28, 4, 128), "bf16", chunks=16, new=(1024, 2048), prefix=(0, 64), lens=3),
        # a handful of chats: a step's weights behind each layer's attention, launches above all
        _case("weights_b8", "weights", (24, 8, 128), "bf16", decodes=8, ctx=(100, 2000), lens=4),
        # Qwen3-Omni thinker shaped decode at full batch
        _case("weights_b256", "weights", (32, 4, 128), "bf16", decodes=256, ctx=(512, 32768), lens=5),
        # prompts that arrive in chunks: every query counts
        _case("weights_chunks", "weights", (28, 4, 128), "bf16", chunks=4, new=(512, 2048), prefix=(0, 8192), lens=6),
        # the last tokens of long prompts look back over an fp8 cache, before it is cut
        _case("weights_observe", "weights", (32, 4, 128), "fp8", chunks=16, new=(32, 32), prefix=(2000, 16384), lens=7),
        # short chats past their budget, one layer at a time
        _case("evict_b8", "evict", (8, 2, 128), "bf16", decodes=8, ctx=(300, 700), keep=256, recent=64, sinks=4, lens=8),
        # one long prompt cut to an eighth in all layers of a 28-layer model
        _case("evict_b1_layers", "evict", (28, 4, 128), "bf16", decodes=1, ctx=(32768, 32768), keep=4096, recent=256, sinks=4,
              layers=28),
        # an Orpheus (Llama-3.2-3B) shaped batch of streams in fp8, some of them still within their budget; 8 layers of it
        _case("evict_b64_fp8", "evict", (24, 8, 128), "fp8", decodes=64, ctx=(500, 4000), keep=1024, recent=128, sinks=4,
              layers=8, lens=9),
        # a full batch of long contexts, a layer of it
        _case("evict_b256", "evict", (32, 4, 128), "bf16", decodes=256, ctx=(512, 32768), keep=2048, recent=256, sinks=16,
              lens=10),
    ]


HEADS = [(8, 2, 128), (24, 8, 128), (32, 4, 128), (28, 4, 128), (8, 1, 256), (16, 2, 256), (16, 4, 64)]
MOST_BYTES, MOST_FLOPS = 2.0e9, 1.5e11


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm_decode", "norm_chunks", "weights_decode", "weights_chunks", "weights_observe", "evict"])
    op = kind.split("_")[0]
    while True:
        heads, kw = rng.choice(HEADS), {"page": rng.choice([16, 16, 16, 32, 64, 128]), "lens": rng.randrange(1 << 20)}
        kw["q"] = rng.choice(["bf16", "bf16", "f16"])
        kv = kw["q"]
        if op == "norm":
            kw.update(rotary=rng.choice([heads[2], heads[2], heads[2] // 2, heads[2] // 4]), interleave=rng.random() < 0.25,
                      llama31=rng.random() < 0.25, theta=rng.choice([1e4, 5e5, 1e6]), first=_log(rng, 1, 200000))
        elif op == "weights":
            kv = rng.choice([kv, kv, "fp8", "mx8", "mx4"])
        else:
            kv = rng.choice([kv, kv, "fp8"])
        if kind == "norm_chunks":
            lo = _log(rng, 1, 1024)
            kw.update(chunks=_log(rng, 1, 16), new=(lo, max(lo, _log(rng, 16, 2048))), prefix=(0, 64))
        elif kind == "norm_decode":
            kw.update(decodes=_log(rng, 1, 512), ctx=(1, 64))
        elif kind == "weights_chunks":
            lo = _log(rng, 1, 1024)
            kw.update(chunks=_log(rng, 1, 8), new=(lo, max(lo, _log(rng, 32, 2048))), prefix=(0, _log(rng, 16, 8192)),
                      causal=rng.random() < 0.75)
        elif kind == "weights_observe":
            n, hi = rng.choice([8, 16, 32, 33, 64]), _log(rng, 256, 16384)
            kw.update(chunks=_log(rng, 1, 32), new=(n, n), prefix=(hi // _log(rng, 1, 16), hi))
        else:
            hi = _log(rng, 64, 32768)
            kw.update(decodes=_log(rng, 1, 256), ctx=(max(1, hi // _log(rng, 1, 64)), hi))
        if op == "evict":
            keep = max(2, hi // _log(rng, 2, 16))
            kw.update(layers=_log(rng, 1, 28), keep=keep, recent=rng.randrange(keep // 2 + 1), sinks=rng.randrange(min(16, keep // 2) + 1))
        c = _case(None, op, heads, kv, **kw)
        w = work(c)
        held = int(_lengths(c)[0].sum()) * c["layers"] * heads[1] * heads[2]
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS and held <= 1.2e9:
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
    n, total = int(new.sum()), int(kv_len.sum())
    row = hkv * d * BITS[case["kv"]] / 8  # K of one cached token
    if case["op"] == "norm":  # q in and out, k and v in and into the cache, positions
        return {"bytes": int(n * (hq * d * 4 + 2 * hkv * d * 2 + 2 * row + 8)), "flops": 0}
    if case["op"] == "weights":  # q and K in, the weights in and out; a product for each visible pair
        at = [np.arange(length - m, length) + 1 if case["causal"] else np.full(m, length) for length, m in zip(kv_len, new)]
        return {"bytes": int(total * row + n * hq * d * 2 + 8 * total * hkv),
                "flops": 2 * d * hq * int(sum(a.sum() for a in at))}
    # weights in, kept ones out with their places; K and V of what moves, which is all but the sinks, in and out
    cut = kv_len > case["keep"]
    kept = np.minimum(kv_len, case["keep"])
    moved = int((kept - case["sinks"])[cut].sum())
    return {"bytes": int(case["layers"] * (4 * moved * row + 4 * hkv * (total + 2 * int(kept.sum())))), "flops": 0}


# ------------------------------------------------------------------ inputs
def _codes(x, kind):
    """(codes, scales) of x [..., head_dim]: blocks scaled so that the largest magnitude is within the codes' range."""
    b = x.float().unflatten(-1, (-1, BLOCK))
    e = torch.floor(torch.log2(b.abs().amax(-1).clamp_min(1e-30))) - (8 if kind == "mx8" else 2)
    y = torch.ldexp(b, -e.unsqueeze(-1).int()).flatten(-2)
    if kind == "mx8":
        codes = y.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    else:  # nearest of 0 0.5 1 1.5 2 3 4 6
        a = y.abs()
        c = sum((a > t).to(torch.uint8) for t in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0))
        c = c | (torch.signbit(y).to(torch.uint8) << 3)
        codes = c[..., 0::2] | (c[..., 1::2] << 4)
    return codes, (e + 127).to(torch.uint8)


def _inputs(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    hq, hkv, d, ps, kind, layers = (case[k] for k in ("q_heads", "kv_heads", "head_dim", "page", "kv", "layers"))
    kv_len, new = _lengths(case)
    pages = -(-kv_len // ps)
    pool = int(pages.sum()) + max(2, int(pages.sum()) // 16)  # the rest of the pool is free or other requests'
    indices = np.random.default_rng(seed).permutation(pool)[: int(pages.sum())].astype(np.int32)
    indptr = np.concatenate([[0], np.cumsum(pages)]).astype(np.int32)
    qo = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    x = {"kv_len": kv_len.tolist(), "new": new.tolist(), "qo": torch.from_numpy(qo), "indptr": torch.from_numpy(indptr),
         "indices": torch.from_numpy(indices), "last": torch.from_numpy((kv_len - (pages - 1) * ps).astype(np.int32)),
         "k_scale": None, "v_scale": None, "scales": None}
    # every request's pages in one row, the shorter ones filled up with the first page
    table = np.zeros((len(pages), max(1, int(pages.max()))), np.int64)
    table[np.arange(table.shape[1])[None] < pages[:, None]] = indices
    x["table"] = torch.from_numpy(table).to(dev)
    x["len"] = torch.from_numpy(kv_len).to(dev)
    x["row_request"] = torch.repeat_interleave(torch.arange(len(new), device=dev), torch.from_numpy(new).to(dev))
    n = int(qo[-1])
    x["at"] = (torch.arange(n, device=dev) - torch.from_numpy(qo[:-1].astype(np.int64)).to(dev)[x["row_request"]]
               + torch.from_numpy(kv_len - new).to(dev)[x["row_request"]])  # each new token's place in its request
    if kind in ("mx8", "mx4"):
        part = torch.empty(pool, 2, ps, hkv, d, device=dev).normal_(generator=g)
        x["kv"], s = _codes(part, kind)
        x["scales"] = s.permute(0, 1, 3, 4, 2).contiguous()
    else:
        x["kv"] = torch.empty(layers, pool, 2, ps, hkv, d, dtype=TORCH[kind], device=dev)
        if kind == "fp8":
            x["k_scale"], x["v_scale"] = (4.5 + torch.rand(2, hkv, device=dev, generator=g)) / 448
        step = max(1, (1 << 28) // (2 * ps * hkv * d))  # pages made at a time
        for layer in range(layers):
            for p in range(0, pool, step):
                part = torch.empty(min(step, pool - p), 2, ps, hkv, d, device=dev).normal_(generator=g)
                if kind == "fp8":
                    part = (part / torch.stack([x["k_scale"], x["v_scale"]]).view(1, 2, 1, hkv, 1)).clamp(-448, 448)
                x["kv"][layer, p:p + part.shape[0]] = part
        if layers == 1:
            x["kv"] = x["kv"][0]
    if case["op"] != "norm":
        # weights as attention leaves them: few heavy tokens, many light ones, some that nothing has looked at
        w = torch.empty(*([layers] if layers > 1 else []), pool, hkv, ps, device=dev).normal_(generator=g)
        x["weights"] = torch.exp(2 * w - 2) * (torch.rand(w.shape, device=dev, generator=g) > 0.02)
    if case["op"] == "norm":
        # q, k and v of one projection, and what the norms learned
        qkv = torch.empty(n, (hq + 2 * hkv) * d, dtype=TORCH[case["q"]], device=dev).normal_(generator=g)
        x["q"], x["k"], x["v"] = (t.unflatten(1, (-1, d)) for t in qkv.split([hq * d, hkv * d, hkv * d], 1))
        x["q_weight"], x["k_weight"] = (1 + 0.2 * torch.empty(2, d, device=dev).normal_(generator=g)).to(TORCH[case["q"]])
        x["pos"] = x["at"] + case["first"]
    elif case["op"] == "weights":
        x["q"] = torch.empty(n, hq, d, dtype=TORCH[case["q"]], device=dev).normal_(generator=g)
    return x


def prepare(case, seed):
    x = _inputs(case, seed)
    s = {"case": case, "x": x}
    if case["op"] == "evict":
        dev = x["weights"].device
        s["on_gpu"] = [x[k].to(dev) for k in ("indptr", "indices", "last")]
        s["out_weights"] = torch.zeros_like(x["weights"])
    if own:
        s["layer"] = x["kv"]
        if x["scales"] is not None:
            from mstar_amd.mx_cache import MXKVLayer

            s["layer"] = MXKVLayer(x["kv"], x["scales"])
        if case["op"] != "evict":
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
    return s


# --------------------------------------------------------------- one pass
def run(s):
    case, x = s["case"], s["x"]
    if own:
        return _own(s, case, x)
    if case["op"] == "norm":
        return _plain_norm(case, x)
    if case["op"] == "evict":
        return _plain_evict(case, x, s["out_weights"])
    return _plain_decode_weights(case, x) if case["chunks"] == 0 else _plain_chunk_weights(case, x)


def _own(s, case, x):
    if case["op"] == "norm":
        s["w"].qk_norm_rope_set_kv_cache(
            s["layer"], x["q"], x["k"], x["v"], x["q_weight"], x["k_weight"], x["pos"], eps=EPS, rotary_dim=case["rotary"],
            interleave=case["interleave"], rope_scale=8 if case["llama31"] else 1, rope_theta=case["theta"], keep_k=False,
            llama31=LLAMA31 if case["llama31"] else None)
        return {"q": x["q"], "kv": x["kv"]}
    if case["op"] == "weights":
        s["w"].accumulate_weights(x["q"], s["layer"], x["weights"], x["k_scale"], x["v_scale"])
        return x["weights"]
    from mstar_amd.eviction import evict_kv_cache

    kept = evict_kv_cache(s["layer"], x["weights"], *s["on_gpu"], keep=case["keep"], recent=case["recent"],
                          sinks=case["sinks"], out_weights=s["out_weights"])
    return {"kept": kept, "kv": x["kv"], "weights": s["out_weights"]}


def _frequencies(case):
    """Each pair's angle a position, in 64 bits."""
    rd = case["rotary"]
    f = case["theta"] ** (-torch.arange(0, rd, 2, dtype=torch.float64) / rd)
    if not case["llama31"]:
        return f
    low, high, old = LLAMA31["low_freq_factor"], LLAMA31["high_freq_factor"], LLAMA31["old_context_len"]
    smooth = ((old * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
    return (1 - smooth) * f / 8 + smooth * f


def _plain_norm(case, x):
    rd = case["rotary"]
    angle = x["pos"].double()[:, None, None] * _frequencies(case).to(x["q"].device)
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()

    def one(t, weight):
        y = t.float()
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.float()
        if case["interleave"]:
            a, b = y[..., 0:rd:2], y[..., 1:rd:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = y[..., : rd // 2], y[..., rd // 2:rd]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([turned, y[..., rd:]], -1)

    x["q"].copy_(one(x["q"], x["q_weight"]))
    page, slot = x["table"][x["row_request"], x["at"] // case["page"]], x["at"] % case["page"]
    x["kv"][page, 0, slot] = one(x["k"], x["k_weight"]).to(x["kv"].dtype)
    x["kv"][page, 1, slot] = x["v"].to(x["kv"].dtype)
    return {"q": x["q"], "kv": x["kv"]}


def _keys(case, x, page, slot):
    """K of cached tokens, [..., kv_heads, head_dim] in 32 bits."""
    rows, kind = x["kv"][page, 0, slot], case["kv"]
    if kind == "fp8":
        return rows.float() * x["k_scale"][:, None]
    if kind not in ("mx8", "mx4"):
        return rows.float()
    if kind == "mx8":
        rows = rows.view(torch.float8_e4m3fn).float()
    else:
        grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=rows.device)
        rows = torch.stack([grid[(rows & 15).int()], grid[(rows >> 4).int()]], -1).flatten(-2)
    scales = x["scales"][page, 0, :, :, slot]
    return torch.ldexp(rows.unflatten(-1, (-1, BLOCK)), scales.int().unsqueeze(-1) - 127).flatten(-2)


def _plain_decode_weights(case, x):
    """All requests at once: their contexts in runs of 256 tokens, a softmax over the runs of a request."""
    dev, run_len, hkv, ps = x["q"].device, 256, case["kv_heads"], case["page"]
    runs = (x["len"] + run_len - 1) // run_len
    request = torch.repeat_interleave(torch.arange(runs.shape[0], device=dev), runs)
    first = torch.arange(request.shape[0], device=dev) - (torch.cumsum(runs, 0) - runs)[request]
    at = first[:, None] * run_len + torch.arange(run_len, device=dev)
    real = at < x["len"][request][:, None]
    at = torch.minimum(at, x["len"][request][:, None] - 1)
    page, slot = x["table"][request[:, None], at // ps], at % ps
    k = _keys(case, x, page, slot).transpose(1, 2).contiguous()  # [runs, kv_heads, 256, head_dim]
    q = x["q"].float().unflatten(1, (hkv, -1)).transpose(2, 3)[request].contiguous()
    p = torch.matmul(k, q) / math.sqrt(case["head_dim"])  # [runs, kv_heads, 256, group]
    p = p.masked_fill(~real[:, None, :, None], -math.inf)
    size = (runs.shape[0], hkv, p.shape[-1])
    top = torch.full(size, -math.inf, device=dev).index_reduce(0, request, p.amax(2), "amax")
    p = torch.exp(p - top[request][:, :, None])
    total = torch.zeros(size, device=dev).index_add(0, request, p.sum(2))
    add = (p / total[request][:, :, None]).sum(-1).transpose(1, 2)  # [runs, 256, kv_heads]
    page, slot, at, add = page[real], slot[real], at[real], add[real]
    last = at == (x["len"][request][:, None] - 1).expand(-1, run_len)[real]
    old = x["weights"][page, :, slot]
    x["weights"][page, :, slot] = torch.where(last[:, None], 0, old) + add
    return x["weights"]


def _plain_chunk_weights(case, x):
    hq, hkv, d, ps = (case[k] for k in ("q_heads", "kv_heads", "head_dim", "page"))
    dev, qo = x["q"].device, x["qo"].tolist()
    for r, (length, n) in enumerate(zip(x["kv_len"], x["new"])):
        at = torch.arange(length, device=dev)
        page, slot = x["table"][r, at // ps], at % ps
        k = _keys(case, x, page, slot).permute(1, 2, 0).contiguous()  # [kv_heads, head_dim, keys]
        q = x["q"][qo[r]:qo[r + 1]].float().unflatten(1, (hkv, -1)).transpose(0, 1).reshape(hkv, -1, d)
        p = torch.matmul(q, k).view(hkv, n, hq // hkv, length) / math.sqrt(d)
        if case["causal"]:
            p = p.masked_fill(at > torch.arange(length - n, length, device=dev)[:, None, None], -math.inf)
        p = torch.exp(p - p.amax(-1, keepdim=True))
        add = (p / p.sum(-1, keepdim=True)).sum((1, 2)).T  # [keys, kv_heads]
        old = x["weights"][page, :, slot]
        x["weights"][page, :, slot] = torch.where((at < length - n)[:, None], old, 0) + add
    return x["weights"]


def _plain_evict(case, x, out_weights):
    """All layers, requests and heads at once, filled up to the longest context."""
    layers, hkv, ps, keep = (case[k] for k in ("layers", "kv_heads", "page", "keep"))
    kv, old, new = (t if layers > 1 else t[None] for t in (x["kv"], x["weights"], out_weights))
    dev, n = kv.device, x["len"].shape[0]
    longest = max(x["kv_len"])
    at = torch.arange(longest, device=dev)
    page, slot = x["table"][:, at // ps], (at % ps).expand(n, -1)
    w = old[:, page, :, slot].permute(2, 0, 3, 1).contiguous()  # [layers, batch, kv_heads, tokens]
    length = x["len"][:, None, None]
    w = w.masked_fill((at < case["sinks"]) | (at >= length - case["recent"]), math.inf)
    w = w.masked_fill(at >= length, -math.inf)
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :keep]
    mine = torch.arange(order.shape[-1], device=dev) < length
    kept = torch.where(mine, order, longest).sort(-1).values
    result = torch.full((layers, n, hkv, keep), -1, dtype=torch.int32, device=dev)
    result[..., : kept.shape[-1]] = torch.where(kept < longest, kept, -1)
    layer, request, head, to = (kept < longest).nonzero(as_tuple=True)
    source = kept[layer, request, head, to]
    from_page, from_slot = x["table"][request, source // ps], source % ps
    to_page, to_slot = x["table"][request, to // ps], to % ps
    rows, values = kv[layer, from_page, :, from_slot, head], old[layer, from_page, head, from_slot]
    kv.view(torch.uint8).view(*kv.shape[:-1], -1)[layer, to_page, :, to_slot, head] = rows.view(torch.uint8)
    new[layer, to_page, head, to_slot] = values
    return {"kept": result if layers > 1 else result[0], "kv": x["kv"], "weights": out_weights}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    x = _inputs(case, seed)
    return {"norm": _exact_norm, "weights": _exact_weights, "evict": _exact_evict}[case["op"]](case, x)


def _exact_norm(case, x):
    rd, ps, d = case["rotary"], case["page"], case["head_dim"]
    pair = np.arange(rd // 2, dtype=np.float64)
    wave = 2 * math.pi * case["theta"] ** (2 * pair / rd)  # positions a turn
    if case["llama31"]:
        lo, hi, old = (LLAMA31[k] for k in ("low_freq_factor", "high_freq_factor", "old_context_len"))
        blend = np.clip((old / wave - lo) / (hi - lo), 0, 1)
        wave = 1 / ((1 - blend) / (8 * wave) + blend / wave)
    turn = torch.from_numpy(x["pos"].cpu().numpy()[:, None] * (2 * math.pi / wave)).to(x["q"].device)
    phase = torch.polar(torch.ones_like(turn), turn)[:, None]

    def rows(t, weight):
        y = t.double()
        y = y / ((y ** 2).sum(-1, keepdim=True) / d + EPS).sqrt() * weight.double()
        pairs = y[..., :rd].unflatten(-1, (-1, 2)) if case["interleave"] else y[..., :rd].unflatten(-1, (2, -1)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * phase)
        y[..., :rd] = z.flatten(-2) if case["interleave"] else z.transpose(-1, -2).flatten(-2)
        return y

    kv = x["kv"].double()
    k, q, t = rows(x["k"], x["k_weight"]), rows(x["q"], x["q_weight"]), 0
    for r, (length, n) in enumerate(zip(x["kv_len"], x["new"])):
        place = np.arange(length - n, length)
        pages, slots = x["table"][r][torch.from_numpy(place // ps)], torch.from_numpy(place % ps)
        kv[pages, 0, slots], kv[pages, 1, slots] = k[t:t + n], x["v"][t:t + n].double()
        t += n
    return {"q": q, "kv": kv}


def _exact_keys(case, x, pages, head):
    """K of one kv head in whole pages, [pages * page, head_dim] in 64 bits."""
    rows = x["kv"][pages, 0, :, head].flatten(0, 1)
    if case["kv"] == "fp8":
        return rows.double() * x["k_scale"][head].double()
    if case["kv"] not in ("mx8", "mx4"):
        return rows.double()
    if case["kv"] == "mx8":
        v = rows.view(torch.float8_e4m3fn).double()
    else:
        both = torch.stack([rows & 15, rows >> 4], -1).flatten(-2).long()
        mag = both & 7
        v = torch.where(mag < 2, mag * 0.5, (1 + (mag & 1) * 0.5) * torch.exp2((mag >> 1).double() - 1))
        v = torch.where(both > 7, -v, v)
    scale = torch.exp2(x["scales"][pages, 0, head].double() - 127)  # [pages, blocks, page]
    return v * scale.transpose(1, 2).flatten(0, 1).repeat_interleave(BLOCK, -1)


def _exact_weights(case, x):
    group, ps = case["q_heads"] // case["kv_heads"], case["page"]
    out, t = x["weights"].double(), 0
    for r, (length, n) in enumerate(zip(x["kv_len"], x["new"])):
        pages = x["table"][r, : -(-length // ps)]
        for h in range(case["kv_heads"]):
            k = _exact_keys(case, x, pages, h)[:length]
            total = torch.zeros(length, dtype=torch.float64, device=k.device)
            for a in range(0, n, 256):  # queries at a time
                b = min(n, a + 256)
                score = x["q"][t + a:t + b, h * group:(h + 1) * group].double().flatten(0, 1) @ k.T * case["head_dim"] ** -0.5
                if case["causal"]:
                    own_place = torch.arange(length - n + a, length - n + b, device=k.device).repeat_interleave(group)
                    score[torch.arange(length, device=k.device)[None] > own_place[:, None]] = -math.inf
                total += torch.softmax(score, -1).sum(0)
            flat = out[pages, h].flatten()
            flat[length - n:length] = 0
            flat[:length] += total
            out[pages, h] = flat.view(-1, ps)
        t += n
    return out


def _exact_evict(case, x):
    layers, hkv, ps, keep = (case[k] for k in ("layers", "kv_heads", "page", "keep"))
    kv, w = ((t if layers > 1 else t[None]) for t in (x["kv"], x["weights"]))
    table, n = x["table"].cpu().numpy(), len(x["kv_len"])
    kept, new = np.full((layers, n, hkv, keep), -1, np.int32), torch.zeros_like(w)
    for r, length in enumerate(x["kv_len"]):
        pages = table[r, : -(-length // ps)]
        on = torch.from_numpy(pages).to(kv.device)
        values = w[:, on].permute(0, 2, 1, 3).flatten(2)[..., :length]  # [layers, kv_heads, tokens]
        host, m = values.cpu().numpy(), min(length, keep)
        choice = np.broadcast_to(np.arange(m), (layers, hkv, m)).copy()
        if length > keep:
            lo, hi = case["sinks"], length - case["recent"]
            best = np.argsort(-host[..., lo:hi], axis=-1, kind="stable")[..., : keep - lo - case["recent"]] + lo
            ends = np.concatenate([np.arange(lo), np.arange(hi, length)])
            choice = np.sort(np.concatenate([best, np.broadcast_to(ends, (layers, hkv, ends.size))], -1), -1)
        kept[:, r, :, :m] = choice
        c = torch.from_numpy(choice).to(kv.device)
        flat = torch.zeros(layers, hkv, on.shape[0] * ps, device=kv.device)
        flat[..., :m] = values.gather(-1, c)
        new[:, on] = flat.unflatten(-1, (-1, ps)).transpose(1, 2)
        if length > keep:
            index = torch.arange(layers, device=kv.device)[:, None, None], torch.arange(hkv, device=kv.device)[:, None]
            rows = kv[index[0], on[c // ps], :, c % ps, index[1]]
            to = torch.arange(m, device=kv.device)
            kv.view(torch.uint8)[index[0], on[to // ps], :, to % ps, index[1]] = rows.view(torch.uint8)
    return {"kept": torch.from_numpy(kept if layers > 1 else kept[0]), "kv": x["kv"], "weights": new if layers > 1 else new[0]}
