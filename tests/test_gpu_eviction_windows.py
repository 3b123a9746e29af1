"""GPU: eviction beside windowed layers, through the cache manager, against 64-bit attention over the whole history."""

import pytest
import torch

from mstar_amd.cache_manager import BatchedCacheManager, WorkspaceBufferManager
from mstar_amd.eviction import kv_weights
from mstar_amd.kv_store import KVCacheConfig, PagedAllocationManager
from oracle import window as W

pytestmark = pytest.mark.gpu

HQ, HKV, D, PS, PAGES = 4, 2, 64, 16, 64
FULL, WINDOWED = 0, 1


def _pool(gpu):
    cfg = KVCacheConfig(num_layers=2, num_kv_heads=HKV, head_dim=D, max_seq_len=1024, max_num_pages=PAGES, page_size=PS, num_qo_heads=HQ)
    kv = torch.zeros(2, PAGES, 2, PS, HKV, D, dtype=torch.bfloat16, device=gpu)
    mgr = PagedAllocationManager(cfg, kv, device=gpu)
    for r in "ab":
        mgr.add_request(r, ["main", "copy"])
    return cfg, kv, mgr, WorkspaceBufferManager(64 << 20, gpu), kv_weights(kv)


def _manager(pool, gpu, rids="ab"):
    """A new one each step, as engines make them: what has been run and cut is known to the pool's allocation manager."""
    cfg, kv, mgr, bufs, weights = pool
    return BatchedCacheManager(list(rids), {r: "main" for r in rids}, kv, mgr, bufs, cfg, gpu, kv_weights=weights)


def _step(pool, gpu, new, g, history, window, sinks, rids="ab"):
    """A full and a windowed layer; the windowed one's output is checked against the whole history."""
    cm = _manager(pool, gpu, rids)
    cm.plan_attention(new)
    for layer in (FULL, WINDOWED):
        x = torch.randn(sum(new), HQ + 2 * HKV, D, generator=g).to(torch.bfloat16)
        q, k, v = x.split([HQ, HKV, HKV], 1)
        call = dict(accumulate=True) if layer == FULL else dict(window_left=window, sink_tokens=sinks)
        out = cm.run_attention(q.to(gpu), k.to(gpu), v.to(gpu), layer_idx=layer, **call).double().cpu()
        if layer == FULL:
            continue
        at = 0
        for r, n in zip(rids, new):
            rows = slice(at, at + n)
            at += n
            kk, vv = history[r] = tuple(torch.cat([old, x_[rows]]) for old, x_ in zip(history[r], (k, v)))
            want, bound = W.attend(q[rows], kk, vv, W.visible(len(kk), n, window, sinks, True), torch.finfo(torch.bfloat16).eps / 2)
            assert ((out[rows] - want).abs() <= bound).all(), (r, n)
    cm.advance_seq_lens()


def _empty():
    return {r: (torch.empty(0, HKV, D, dtype=torch.bfloat16),) * 2 for r in "ab"}


@pytest.mark.parametrize("window,sinks", [(0, 0), (15, 0), (16, 3), (20, 2)])
def test_windows_are_exact_behind_an_eviction(gpu, window, sinks):
    """As many last and first tokens kept as the window and its sinks span, no more: every later step sees what it would have seen."""
    pool, g, history = _pool(gpu), torch.Generator().manual_seed(1), _empty()
    _step(pool, gpu, [100, 30], g, history, window, sinks)
    for keep, then in ((40, ([1, 1], [1, 1], [9, 2])), (33, ([1, 1], [30, 1]))):
        _manager(pool, gpu).evict(keep, recent=window, sinks=sinks)
        for new in then:
            _step(pool, gpu, new, g, history, window, sinks)


def test_evictions_that_would_cut_into_a_window_are_refused(gpu):
    pool, g, history = _pool(gpu), torch.Generator().manual_seed(1), _empty()
    _step(pool, gpu, [100, 30], g, history, 20, 2)
    kv, weights = pool[1].clone(), pool[4].clone()
    for bad in (dict(recent=19, sinks=2), dict(recent=20, sinks=1), dict(), dict(recent=40)):
        with pytest.raises(ValueError, match="window"):
            _manager(pool, gpu).evict(40, **bad)
    assert torch.equal(kv, pool[1]) and torch.equal(weights, pool[4])
    assert pool[2].get_state("a", "main").seq_len == 100 and not pool[2].get_state("a", "main").evicted
    assert _manager(pool, gpu).evict(40, recent=20, sinks=2) == 4


def test_windows_past_what_an_eviction_left_are_refused(gpu):
    """A layer first run with a window, or a longer one, behind the eviction: refused for requests that were cut, before the append."""
    pool, g = _pool(gpu), torch.Generator().manual_seed(1)
    cm = _manager(pool, gpu)

    def run(new, rids="ab", **call):
        cm = _manager(pool, gpu, rids)
        cm.plan_attention(new)
        q, k, v = torch.randn(sum(new), HQ + 2 * HKV, D, generator=g).to(torch.bfloat16).to(gpu).split([HQ, HKV, HKV], 1)
        kv, q0 = pool[1].clone(), q.clone()
        try:
            cm.run_attention(q, k, v, layer_idx=0, **call)
        except ValueError:
            cm.plan_rope(new)
            with pytest.raises(ValueError, match="window"):
                cm.apply_rope_and_run_attention(q, k, v, layer_idx=0, **call)
            assert torch.equal(pool[1], kv) and torch.equal(q, q0)
            raise
        cm.advance_seq_lens()

    run([100, 30], accumulate=True)
    assert cm.evict(40, recent=10, sinks=1) == 4  # of a alone
    for bad in (dict(window_left=11), dict(window_left=10, sink_tokens=2), dict(window_left=500)):
        with pytest.raises(ValueError, match="window"):
            run([1, 1], **bad)
        run([1], "b", **bad)  # was not cut
    pool[2].windows = (-1, 0)
    run([1, 1], window_left=10, sink_tokens=1)
    run([1, 1])
