"""Pools beyond 4 GiB: the serving operators on pages at the far end of one give what they give in a small one, bit for bit.
(Whole numbers and bytes: equal. The outputs: the same sums in the same order, so equal too.)"""
import numpy as np
import pytest

from test_gpu_decode import setup

pytestmark = pytest.mark.gpu


def test_pages_past_32_bit_offsets(yahkv, torch_gpu):
    torch = torch_gpu
    lens, budget, pt, n_kv, hd = [700, 65, 333], 64, 64, 4, 256
    g, table, host, dev, rng = setup(yahkv, torch, 8, 24, n_kv, hd, pt, lens, seed=9)
    small_n = dev.geom.n_pages
    P = 2 ** 32 // (pt * hd * n_kv) + 2 * small_n                       # 64 KiB of K codes a page: the last lie past 4 GiB
    far = yahkv.DevicePools(yahkv.geometry(8, 24, n_kv, hd, pt, P))
    near = yahkv.DevicePools(yahkv.geometry(8, 24, n_kv, hd, pt, 2 * small_n))
    for name in ("kq", "ks", "vq", "vs"):
        a, b, c = getattr(dev, name), getattr(far, name), getattr(near, name)
        b[-2 * a.numel():-a.numel()].copy_(a), c[:a.numel()].copy_(a)
    t = lambda x: torch.from_numpy(np.ascontiguousarray(x.astype(np.int32))).cuda()
    seq_len = t(np.array(lens))
    q = torch.randn(3, 24, hd, device="cuda").half()
    rotary = yahkv.Rotary(64, 1e4)
    k, v = torch.randn(3, 9, n_kv, hd, device="cuda").half(), torch.randn(3, 9, n_kv, hd, device="cuda").half()
    new = np.arange(small_n, small_n + 3).reshape(3, 1)                  # fresh pages behind the sequences' own
    results = []
    for pools, base in ((near, 0), (far, P - 2 * small_n)):
        tab, fresh = t(table + base), t(new + base)
        shared = yahkv.decode_attend_shared(pools, tab, seq_len, t(np.array([0, 1, 2, 3])), t(np.array([640, 64, 320])), 640, 700, q, 0.0625)
        w = torch.zeros(3, n_kv, 704, device="cuda")
        out = yahkv.decode_attend_weights(pools, tab, seq_len, 700, q, 0.0625, w)
        kept, n_kept = yahkv.evict_select(pools.geom, seq_len, 700, w, budget - 9, 4, 8)
        yahkv.evict_compact(pools, tab, kept, n_kept, fresh)
        yahkv.rotary_append(pools, fresh, n_kept, rotary, k, v)
        end = yahkv.decode_attend(pools, fresh, n_kept + 9, budget, q, 0.0625)
        tail = [getattr(pools, name)[-getattr(dev, name).numel():] for name in ("kq", "ks", "vq", "vs")]
        results.append([shared, out, w, kept, n_kept, end, *tail])
    for i, (a, b) in enumerate(zip(*results)):
        assert torch.equal(a, b), i
    assert bool(results[0][0].isfinite().all()) and bool(results[0][5].isfinite().all())
