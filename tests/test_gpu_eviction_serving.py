"""GPU: norm + rotate + append, attention, accumulated weights and eviction together, through the cache manager.

Requests prefill, decode, are cut to a budget and go on; at every step the cache's rows, the attention
over them, the weights and what an eviction keeps are compared with 64 bits.
"""

import numpy as np
import pytest
import torch

from gpu_helpers import log
from mstar_amd.cache_manager import BatchedCacheManager, WorkspaceBufferManager
from mstar_amd.eviction import kv_weights
from mstar_amd.kv_store import KVCacheConfig, PagedAllocationManager
from mstar_amd.mx_cache import MXKVCache, read_kv_cache
from oracle import eviction as E
from oracle import qk_norm as N
from oracle import window as W

pytestmark = pytest.mark.gpu

HQ, HKV, D, PS, PAGES, LAYERS = 8, 2, 128, 16, 200, 2
ROPE = dict(rotary_dim=D, interleave=False, rope_scale=1.0, rope_theta=1e6, llama31=None)
CALL = dict(rotary_dim=D, interleave=False, rope_scale=1.0, rope_theta=1e6)


def _manager(gpu, kind, weights=True):
    cfg = KVCacheConfig(num_layers=LAYERS, num_kv_heads=HKV, head_dim=D, max_seq_len=4096, max_num_pages=PAGES, page_size=PS,
                        num_qo_heads=HQ)
    if kind == "mx8":
        kv = MXKVCache(LAYERS, PAGES, PS, HKV, D, bits=8, device=gpu)
    else:
        kv = torch.zeros(LAYERS, PAGES, 2, PS, HKV, D, dtype=torch.bfloat16, device=gpu)
    mgr = PagedAllocationManager(cfg, None if kind == "mx8" else kv, device=gpu)
    rids = ["a", "b", "c"]
    for i, r in enumerate(rids):
        mgr.add_request(r, ["main", "copy"])
        mgr.get_state(r, "main").position_id_start = 1000 * i
    # NaN weights: no slot may count before its token's step has written it
    w = kv_weights(kv).fill_(float("nan")) if weights else None
    return BatchedCacheManager(rids, {r: "main" for r in rids}, kv, mgr, WorkspaceBufferManager(64 << 20, gpu), cfg, gpu, kv_weights=w)


def _context(cm, rid, layer, label="main"):
    """K, V [tokens, heads, d] in float64 and weights [tokens, heads] of a request as they are now."""
    st = cm._get_state(rid, label)
    n = -(-st.seq_len // PS)
    idx = (torch.tensor([0, n], dtype=torch.int32), torch.tensor(st.page_indices[:n], dtype=torch.int32),
           torch.tensor([st.seq_len - (n - 1) * PS], dtype=torch.int32))
    k, v = read_kv_cache(cm.kv_cache[layer], *idx, st.seq_len, dtype=torch.float32)
    w = cm.kv_weights[layer][torch.tensor(st.page_indices[:n], device=cm.device)].transpose(1, 2).flatten(0, 1)[: st.seq_len]
    return k.double().cpu(), v.double().cpu(), w.double().cpu()


@pytest.mark.parametrize("kind", ["bf16", "mx8"])
def test_a_run_of_steps(gpu, kind):
    cm = _manager(gpu, kind)
    g = torch.Generator().manual_seed(4)
    weights = [tuple((1 + 0.2 * torch.randn(D, generator=g)).to(torch.bfloat16) for _ in range(2)) for _ in range(LAYERS)]
    total = [0, 0, 0]  # tokens a request has been given
    # prompts, steps, cut, steps (one request a chunk), cut again
    script = [[200, 37, 90], [1, 1, 1], [1, 1, 1], "cut", [1, 1, 1], [40, 1, 1], "cut", [1, 1, 1]]
    keep, recent, sinks = 48, 16, 2
    for at, step in enumerate(script):
        if step == "cut":
            before = {(r, l): _context(cm, r, l) for r in cm.request_ids for l in range(LAYERS)}
            pages = {r: len(cm._get_state(r).page_indices) for r in cm.request_ids}
            free = cm.alloc_manager.num_free_pages
            freed = cm.evict(keep, recent=recent, sinks=sinks)
            assert freed == sum(max(0, p - 3) for p in pages.values()) and cm.alloc_manager.num_free_pages == free + freed > free
            for (r, l), (k, v, w) in before.items():
                st = cm._get_state(r)
                n = min(k.shape[0], keep)
                assert st.seq_len == n and len(st.page_indices) == min(pages[r], 3)
                k2, v2, w2 = _context(cm, r, l)
                for h in range(HKV):
                    places = torch.as_tensor(E.kept_places(w[:, h].float().numpy(), keep, recent, sinks))
                    assert torch.equal(k2[:, h], k[places, h]) and torch.equal(v2[:, h], v[places, h]) and torch.equal(w2[:, h], w[places, h])
            continue
        t = sum(step)
        cm.plan_attention(step)
        cm.plan_rope(step)
        for l in range(LAYERS):
            held = [_context(cm, r, l) if cm._get_state(r).seq_len else None for r in cm.request_ids]
            x = torch.randn(t, HQ + 2 * HKV, D, generator=g).to(torch.bfloat16)
            q, k, v = x.to(gpu).split([HQ, HKV, HKV], 1)
            out = cm.apply_rope_and_run_attention(q, k, v, layer_idx=l, q_norm_weight=weights[l][0].to(gpu),
                                                  k_norm_weight=weights[l][1].to(gpu), norm_eps=1e-6, accumulate=True, **CALL)
            torch.cuda.synchronize()
            row = 0
            for i, (r, n) in enumerate(zip(cm.request_ids, step)):
                rows = slice(row, row + n)
                row += n
                st = cm._get_state(r)
                length = st.seq_len + n
                st.seq_len = length  # as it will be
                ck, cv, cw = _context(cm, r, l)
                st.seq_len = length - n
                if held[i] is not None:  # what was there is as it was
                    assert torch.equal(ck[:-n], held[i][0]) and torch.equal(cv[:-n], held[i][1])
                pos = torch.arange(n) + total[i] + 1000 * i  # positions go on as if nothing had been cut
                want, bound = N.norm_rope(x[rows, HQ:HQ + HKV], weights[l][1], pos, 1e-6, **ROPE)
                if kind == "bf16":
                    assert ((ck[-n:] - want).abs() <= N.rounded(want, bound, torch.bfloat16)).all()
                else:
                    peak = (want.abs() + bound).unflatten(-1, (-1, 32)).amax(-1, keepdim=True).expand(n, HKV, D // 32, 32).flatten(-2)
                    assert ((ck[-n:] - want).abs() <= bound + (want.abs() + bound) * 2.0 ** -4 + peak * 2.0 ** -10 * 4 / 464).all()
                qr, qb = N.norm_rope(x[rows, :HQ], weights[l][0], pos, 1e-6, **ROPE)
                got_q = q[rows].cpu()
                assert ((got_q.double() - qr).abs() <= N.rounded(qr, qb, torch.bfloat16)).all()
                seen = W.visible(length, n, -1, 0, True)
                o, ob = W.attend(got_q, ck, cv, seen, torch.finfo(torch.bfloat16).eps / 2)
                assert ((out[rows].double().cpu() - o).abs() <= ob + 1e-30).all(), (at, l, r)
                add, ab = E.probabilities(got_q, ck, seen)
                if held[i] is not None:
                    add[:-n] += held[i][2]
                assert ((cw - add).abs() <= ab + add.abs() * 2.0 ** -23).all(), (at, l, r)
        cm.advance_seq_lens()
        total = [a + n for a, n in zip(total, step)]
        log(f"{kind} step {at}: lengths {[cm._get_state(r).seq_len for r in cm.request_ids]}")
    assert [cm._get_state(r).position_id_start for r in cm.request_ids] == [a + 1000 * i for i, a in enumerate(total)]


def test_a_request_named_twice_is_cut_once(gpu):
    cm = _manager(gpu, "bf16")
    g = torch.Generator().manual_seed(9)
    cm.plan_attention([100, 60, 20])
    for l in range(LAYERS):
        x = torch.randn(180, HQ + 2 * HKV, D, generator=g).to(torch.bfloat16).to(gpu)
        cm.run_attention(*x.split([HQ, HKV, HKV], 1), layer_idx=l, accumulate=True)
    cm.advance_seq_lens()
    before = {(r, l): _context(cm, r, l) for r in cm.request_ids for l in range(LAYERS)}
    cm.request_ids = ["a", "b", "a"]
    free = cm.alloc_manager.num_free_pages
    assert cm.evict(32, recent=8, sinks=2) == (7 - 2) + (4 - 2) and cm.alloc_manager.num_free_pages == free + 7
    assert [cm._get_state(r).seq_len for r in "abc"] == [32, 32, 20]
    for (r, l), (k, v, w) in before.items():
        got = _context(cm, r, l)
        for h in range(HKV):
            places = torch.as_tensor(E.kept_places(w[:, h].float().numpy(), 32, 8, 2))
            assert all(torch.equal(a[:, h], b[places, h]) for a, b in zip(got, (k, v, w)))


@pytest.mark.parametrize("kind", ["bf16", "mx8"])
def test_snapshot_of_a_cut_request(gpu, kind):
    """A copy of a cut request holds its rows and weights, also over a copy that was made before the cut."""
    cm = _manager(gpu, kind)
    g = torch.Generator().manual_seed(4)
    qw, kw = (torch.ones(D, dtype=torch.bfloat16, device=gpu) for _ in range(2))

    def step(lens):
        cm.plan_attention(lens)
        cm.plan_rope(lens)
        for l in range(LAYERS):
            x = torch.randn(sum(lens), HQ + 2 * HKV, D, generator=g).to(torch.bfloat16).to(gpu)
            cm.apply_rope_and_run_attention(*x.split([HQ, HKV, HKV], 1), layer_idx=l, q_norm_weight=qw, k_norm_weight=kw,
                                            accumulate=True, **CALL)
        cm.advance_seq_lens()

    step([60, 20, 33])
    cm.snapshot_all("main", "copy")
    cm.evict(40, recent=4)
    step([20, 40, 27])  # as long as it was: 60 tokens, of which only the places are the copy's
    cm.snapshot_all("main", "copy")
    torch.cuda.synchronize()
    for r in cm.request_ids:
        for l in range(LAYERS):
            for a, b in zip(_context(cm, r, l), _context(cm, r, l, "copy")):
                assert torch.equal(a, b)


def test_norm_then_run_is_the_fused_call(gpu):
    """apply_qk_norm_rope then run_attention gives what apply_rope_and_run_attention with norms gives, bit for bit."""
    a, b = _manager(gpu, "bf16"), _manager(gpu, "bf16")
    g = torch.Generator().manual_seed(4)
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=g)).to(gpu) for _ in range(2))  # fp32 weights
    for step in ([30, 1, 7], [1, 1, 1]):
        x = torch.randn(sum(step), HQ + 2 * HKV, D, generator=g).to(torch.bfloat16).to(gpu)
        outs = []
        for cm, fused in ((a, True), (b, False)):
            cm.plan_attention(step)
            cm.plan_rope(step)
            q, k, v = x.clone().split([HQ, HKV, HKV], 1)
            if fused:
                outs.append(cm.apply_rope_and_run_attention(q, k, v, q_norm_weight=qw, k_norm_weight=kw, norm_eps=1e-5, accumulate=True, **CALL))
            else:
                q, k = cm.apply_qk_norm_rope(q, k, qw, kw, eps=1e-5, **CALL)
                outs.append(cm.run_attention(q, k, v, accumulate=True))
            cm.advance_seq_lens()
        assert torch.equal(*outs) and torch.equal(a.kv_cache, b.kv_cache)
        assert torch.equal(a.kv_weights.view(torch.int32), b.kv_weights.view(torch.int32))


def test_manager_refusals(gpu):
    cm = _manager(gpu, "bf16", weights=False)
    with pytest.raises(ValueError):
        cm.evict(10)
    step = [5, 1, 2]
    cm.plan_attention(step)
    cm.plan_rope(step)
    q, k, v = torch.zeros(8, HQ + 2 * HKV, D, dtype=torch.bfloat16, device=gpu).split([HQ, HKV, HKV], 1)
    w = torch.ones(D, device=gpu)
    with pytest.raises(ValueError):
        cm.apply_rope_and_run_attention(q, k, v, q_norm_weight=w)
    with pytest.raises(ValueError):
        cm.run_attention(q, k, v, accumulate=True)
    cm.kv_weights = kv_weights(cm.kv_cache)
    with pytest.raises(ValueError):
        cm.run_attention(q, k, v, accumulate=True, window_left=3)
    for bad in (dict(keep=0), dict(keep=5, recent=6), dict(keep=5, recent=3, sinks=3), dict(keep=5, sinks=-1)):
        with pytest.raises(ValueError):
            cm.evict(**bad)
    assert cm.evict(100) == 0
    with pytest.raises(ValueError):
        BatchedCacheManager(cm.request_ids, cm.active_labels, cm.kv_cache, cm.alloc_manager, cm.buffer_manager, cm.kv_cache_config, gpu,
                            kv_weights=torch.zeros(1, PAGES, HKV, PS, device=gpu))
