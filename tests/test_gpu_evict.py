"""Eviction by accumulated attention weight: the weights against float64, the choice and the move against plain indexing (whole
numbers and bytes: equal), and the run of them with rotary positions and shared prefixes as a serving loop has it.

Tolerance of a weight, in u = 2^-24: a score is a sum of 256 exact products at most, 32 at a time, whose f32 sums err by at most
48 u sum |q k| scale (32 inside a block, 8 blocks, the scale's products), so a numerator by that times e, and the denominator,
a sum of positive terms in a tree of at most 64 sequential steps, by the largest of those and 64 u: relative 2 x 48 u x (largest
sum |q k| scale of the row) + 128 u, and half a step of the running sum it is added to."""
import numpy as np
import pytest

import oracle
from helpers import dequant, logical_blocks, make_tables
from test_gpu_decode import closed, setup
from test_gpu_shared import check

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def exact_weights(g, table, host, lens, q, scale):
    """(weights [n][H][T], relative tolerance [n][H]) in float64."""
    G = g.n_q_heads // g.n_kv_heads
    T = max(max(lens), 1)
    w, tol = np.zeros((len(lens), g.n_kv_heads, T)), np.zeros((len(lens), g.n_kv_heads))
    for s, n in enumerate(lens):
        if n == 0:
            continue
        (ks, kc), _ = logical_blocks(host.arrays(), g, table[s], n)
        k = dequant(ks, kc).astype(np.float64)
        for h in range(g.n_kv_heads):
            x = q[s, h * G:(h + 1) * G] @ k[:, h].T * scale
            p = np.exp(x - x.max(-1, keepdims=True))
            w[s, h, :n] = (p / p.sum(-1, keepdims=True)).sum(0)
            tol[s, h] = 2 * 48 * U * (np.abs(q[s, h * G:(h + 1) * G]) @ np.abs(k[:, h]).T * scale).max() + 128 * U
    return w, tol


@pytest.mark.parametrize("fmt,n_q,n_kv,hd,pt,lens", [
    (8, 24, 4, 256, 64, [700, 1, 0, 64, 65, 333]), (4, 32, 8, 128, 16, [100, 0, 2000, 17]), (8, 8, 1, 256, 32, [1]),
    (4, 8, 8, 128, 64, [63, 129]), (8, 3, 1, 128, 16, [5000, 15]), (8, 24, 4, 256, 64, [9000]), (4, 24, 4, 256, 32, [0, 0])])
def test_weights(yahkv, torch_gpu, fmt, n_q, n_kv, hd, pt, lens):
    torch = torch_gpu
    g, table, host, dev, rng = setup(yahkv, torch, fmt, n_q, n_kv, hd, pt, lens, seed=hd + len(lens), fill=0x7F)
    n, T, scale = len(lens), max(max(lens), 1), hd ** -0.5
    q = torch.from_numpy(rng.standard_normal((n, n_q, hd)).astype(np.float32)).cuda().to(torch.bfloat16)
    gate = torch.randn(n, n_q, hd, device="cuda")
    t_table, t_len = torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    want, rel = exact_weights(g, table, host, lens, q.double().cpu().numpy(), scale)
    out_want = closed(g, table, host, lens, q.double().cpu().numpy(), scale, gate.double().cpu().numpy())
    w = torch.full((n, n_kv, T + 3), -7.0, device="cuda")
    out = yahkv.decode_attend_weights(dev, t_table, t_len, T, q, scale, w, gate=gate, out_dtype=torch.float16)
    if max(lens):
        check(torch, out, out_want, torch.float16)
    else:
        assert not out.any()
    got = w.double().cpu().numpy()
    for s, m in enumerate(lens):
        assert np.all(np.abs(got[s, :, :m] - want[s, :, :m]) <= want[s, :, :m] * rel[s][:, None] + 2.0 ** -149)
        assert np.all(got[s, :, m:] == -7.0)                                   # behind the length: left alone
        # half a step of each of up to 8 rows' sums besides, over m keys
        assert m == 0 or np.all(np.abs(got[s, :, :m].sum(-1) - n_q // n_kv) <= (n_q // n_kv) * (rel[s] + 16 * U))
    # added to what was there, with decay, in place and out of place
    base = torch.rand(n, n_kv, T + 3, device="cuda") * 3
    other = torch.zeros_like(base)
    yahkv.decode_attend_weights(dev, t_table, t_len, T, q, scale, other, weights_in=base, decay=0.5)
    b64 = base.double().cpu().numpy()
    yahkv.decode_attend_weights(dev, t_table, t_len, T, q, scale, base, weights_in=base, decay=0.5)
    for s, m in enumerate(lens):
        total = 0.5 * b64[s, :, :m] + want[s, :, :m]
        for x in (other, base):
            assert np.all(np.abs(x[s, :, :m].double().cpu().numpy() - total) <= want[s, :, :m] * rel[s][:, None] + total * 2 * U)
        assert torch.equal(other[s, :, m:], torch.zeros_like(other[s, :, m:]))
        assert np.array_equal(base[s, :, m:].double().cpu().numpy(), b64[s, :, m:])


@pytest.mark.parametrize("fmt,n_q,n_kv,hd,pt", [
    (8, 24, 4, 256, 64), (8, 8, 1, 256, 32), (8, 6, 3, 256, 16), (8, 32, 8, 128, 64), (8, 10, 5, 128, 32), (8, 4, 2, 128, 16),
    (4, 8, 1, 256, 64), (4, 24, 4, 256, 32), (4, 16, 8, 256, 16), (4, 6, 3, 128, 64), (4, 3, 1, 128, 32), (4, 32, 8, 128, 16)])
def test_weights_of_a_large_batch(yahkv, torch_gpu, fmt, n_q, n_kv, hd, pt):
    """The form for batches of more tiles than waves hold (a partial per wave, the line cut by tile where the kv heads divide
    eight): the host's bound alone asks for it, the lengths stay short."""
    torch = torch_gpu
    lens = [700, 1, 0, 64, 65, 333, 2000, 17, 0, 130]
    g, table, host, dev, rng = setup(yahkv, torch, fmt, n_q, n_kv, hd, pt, lens, seed=hd + pt + n_kv, fill=0x7F)
    n, T, bound, scale = len(lens), max(lens), 70001, hd ** -0.5
    q = torch.from_numpy(rng.standard_normal((n, n_q, hd)).astype(np.float32)).cuda().to(torch.bfloat16)
    t_table, t_len = torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    want, rel = exact_weights(g, table, host, lens, q.double().cpu().numpy(), scale)
    out_want = closed(g, table, host, lens, q.double().cpu().numpy(), scale)
    base = torch.rand(n, n_kv, bound + 2, device="cuda") * 3
    b64 = base[:, :, :T].double().cpu().numpy()
    w = base.clone()
    out = yahkv.decode_attend_weights(dev, t_table, t_len, bound, q, scale, w, weights_in=w, decay=0.5)
    check(torch, out, out_want, torch.float32)
    got = w[:, :, :T].double().cpu().numpy()
    for s, m in enumerate(lens):
        total = 0.5 * b64[s, :, :m] + want[s, :, :m]
        assert np.all(np.abs(got[s, :, :m] - total) <= want[s, :, :m] * rel[s][:, None] + total * 2 * U), s
        assert torch.equal(w[s, :, m:], base[s, :, m:])                        # behind the length: left alone
        assert m > 0 or not out[s].any()


@pytest.mark.parametrize("fmt,n_q,n_kv,hd,pt,bound", [(8, 24, 4, 256, 64, 0), (8, 24, 4, 256, 64, 70001), (4, 32, 8, 128, 16, 0),
                                                      (8, 8, 1, 256, 32, 70001), (4, 6, 3, 128, 64, 70001)])
def test_weights_of_scores_far_from_zero(yahkv, torch_gpu, fmt, n_q, n_kv, hd, pt, bound):
    """Scores of 1e9, where a unit of their last place is 64: a row's largest has all of its weight (the others are millions
    below it), and a key's weights are a whole number."""
    torch = torch_gpu
    lens = [700, 1, 0, 64, 65, 333, 2000, 17, 130]
    g, table, host, dev, rng = setup(yahkv, torch, fmt, n_q, n_kv, hd, pt, lens, seed=hd + pt + n_kv, fill=0x7F)
    n, T, scale = len(lens), max(lens), hd ** -0.5
    ks = dev.ks.view(torch.float16)
    ks.copy_(torch.where(torch.isfinite(ks), torch.full_like(ks, 32768.0), ks))
    for name, arr in host.arrays().items():
        arr.reshape(-1)[:] = dev.numpy()[name].reshape(-1)
    q = torch.from_numpy(200 * rng.standard_normal((n, n_q, hd)).astype(np.float32)).cuda().half()
    want, _ = exact_weights(g, table, host, lens, q.double().cpu().numpy(), scale)
    assert np.all(np.abs(want - np.round(want)) < 1e-9)
    w = torch.full((n, n_kv, (bound or T) + 2), -1.0, device="cuda")
    out = yahkv.decode_attend_weights(dev, torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), bound or T, q,
                                      scale, w)
    check(torch, out, closed(g, table, host, lens, q.double().cpu().numpy(), scale), torch.float32)
    for s, m in enumerate(lens):
        assert np.array_equal(w[s, :, :m].double().cpu().numpy(), np.round(want[s, :, :m])), s
        assert bool((w[s, :, m:] == -1.0).all())


def test_weights_from_a_graph(yahkv, torch_gpu):
    torch = torch_gpu
    lens = [700, 64, 0, 333]
    g, table, host, dev, rng = setup(yahkv, torch, 8, 24, 4, 256, 64, lens, seed=3)
    t_table, t_len = torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn(4, 24, 256, device="cuda").half()
    w, out = torch.zeros(4, 4, 704, device="cuda"), torch.empty(4, 24, 256, device="cuda")
    ws = torch.empty(yahkv.decode_weights_workspace_bytes(dev.geom, 4, 700), dtype=torch.uint8, device="cuda")
    step = lambda: yahkv.decode_attend_weights(dev, t_table, t_len, 700, q, 0.0625, w, weights_in=w, out=out, workspace=ws)
    step()
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            step()
    for i in range(3):
        q.copy_(torch.randn(4, 24, 256, device="cuda"))
        w.zero_()
        step()
        want, o = w.clone(), out.clone()
        w.zero_(), out.fill_(float("nan")), ws.random_(0, 256)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(w, want) and torch.equal(out, o), i


def select_plain(w, lens, budget, sink, recent):
    n, H, _ = w.shape
    kept = np.full((n, H, budget), -1, np.int32)
    for s in range(n):
        m = int(lens[s])
        for h in range(H):
            if m <= budget:
                kept[s, h, :m] = np.arange(m)
                continue
            x = np.where(w[s, h, :m] > 0, w[s, h, :m], 0.0)
            mid = np.arange(sink, m - recent)
            best = mid[np.argsort(-x[mid], kind="stable")[:budget - sink - recent]]
            kept[s, h] = np.sort(np.concatenate([np.arange(sink), best, np.arange(m - recent, m)]))
    return kept


@pytest.mark.parametrize("kind", ["normal", "ties", "zeros", "odd"])
@pytest.mark.parametrize("budget,sink,recent", [(1, 0, 0), (1, 1, 0), (8, 4, 4), (64, 4, 16), (257, 0, 100), (1000, 1, 0), (5000, 4, 512)])
def test_select(yahkv, torch_gpu, budget, sink, recent, kind):
    torch = torch_gpu
    rng = np.random.default_rng(budget + len(kind))
    lens = np.array([0, 1, budget - 1, budget, budget + 1, 63, 64, 65, 1023, 1025, 4099, 9000])
    T = 9005
    g = yahkv.geometry(8, 8, 2, 128, 16, 4)
    w = np.exp(rng.standard_normal((len(lens), 2, T)) * 3).astype(np.float32)
    if kind == "ties":
        w = np.floor(w).astype(np.float32)
    elif kind == "zeros":
        w[:] = 0.0
    elif kind == "odd":                                               # NaN, infinities, negative and subnormal values
        w[..., ::7], w[..., 3::11], w[..., 5::13], w[..., 1::17] = np.nan, np.inf, -3.0, 1e-40
        w[..., 2::19] = -0.0
    kept, n_kept = yahkv.evict_select(g, torch.tensor(lens, dtype=torch.int32, device="cuda"), T, torch.from_numpy(w).cuda(), budget, sink, recent)
    with np.errstate(invalid="ignore"):
        assert np.array_equal(kept.cpu().numpy(), select_plain(w, lens, budget, sink, recent))
    assert np.array_equal(n_kept.cpu().numpy(), np.minimum(lens, budget))


@pytest.mark.parametrize("length,budget", [(32768, 4096), (32769, 1), (70001, 60000), (200000, 777)])
def test_select_long(yahkv, torch_gpu, length, budget):
    torch = torch_gpu
    g = yahkv.geometry(8, 8, 2, 128, 16, 4)
    w = torch.rand(1, 2, length + 1, device="cuda")
    w[0, 1] = torch.floor(w[0, 1] * 8)
    lens = torch.tensor([length], dtype=torch.int32, device="cuda")
    kept, _ = yahkv.evict_select(g, lens, length + 1, w, budget, 0, min(64, budget - 1))
    assert np.array_equal(kept.cpu().numpy(), select_plain(w.cpu().numpy(), [length], budget, 0, min(64, budget - 1)))
    clamped, n = yahkv.evict_select(g, lens, length - 5, w, budget, 0, 0)           # lengths beyond the host's bound are cut
    assert np.array_equal(clamped.cpu().numpy(), select_plain(w.cpu().numpy(), [length - 5], budget, 0, 0))
    assert int(n[0]) == min(budget, length - 5)


@pytest.mark.parametrize("fmt,n_kv,hd,pt", [(8, 4, 256, 64), (8, 2, 128, 16), (4, 4, 256, 32), (4, 8, 128, 64), (8, 1, 128, 32), (4, 1, 256, 16)])
@pytest.mark.parametrize("budget", [1, 16, 100, 129])
def test_compact(yahkv, torch_gpu, fmt, n_kv, hd, pt, budget):
    """Codes and scales moved bit for bit, weights along, everything else in the pools as it was."""
    torch = torch_gpu
    rng = np.random.default_rng(budget + hd + pt)
    lens = [400, 0, 1, budget, budget + 1, 90]
    need = [(n + pt - 1) // pt for n in lens]
    new = (budget + pt - 1) // pt
    P = sum(need) + new * len(lens) + 1
    g = yahkv.geometry(fmt, n_kv * 2, n_kv, hd, pt, P)
    perm = rng.permutation(P).astype(np.int32)
    table = make_tables(rng, need, sum(need))
    table = perm[:sum(need)][table]
    dst = perm[sum(need):sum(need) + new * len(lens)].reshape(len(lens), new)
    b = yahkv.pool_bytes(g)
    arrays = {k: rng.integers(0, 256, b[k], dtype=np.uint8) for k in b}
    dev = yahkv.DevicePools(g)
    dev.load(arrays)
    w = rng.random((len(lens), n_kv, 400)).astype(np.float32)
    t = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()
    kept, n_kept = yahkv.evict_select(g, t(np.array(lens, np.int32)), 400, t(w), budget)
    w_out = torch.full((len(lens), n_kv, budget + 2), -1.0, device="cuda")
    yahkv.evict_compact(dev, t(table), kept, n_kept, t(dst), t(w), w_out)
    kept, NB, kb = kept.cpu().numpy(), hd // 32, 32 if fmt == 8 else 16
    kq, ks = arrays["kq"].reshape(P, n_kv, NB, pt, kb), arrays["ks"].view(np.uint16).reshape(P, n_kv, pt, NB)
    vq, vs = arrays["vq"].reshape(P, n_kv, -1, pt), arrays["vs"].view(np.uint16).reshape(P, n_kv, NB, pt)
    want_w = np.full((len(lens), n_kv, budget + 2), -1.0, np.float32)
    for s, n in enumerate(lens):
        for h in range(n_kv):
            for i in range(min(n, budget)):
                a, b2 = kept[s, h, i] // pt, kept[s, h, i] % pt
                p, d, j = table[s, a], dst[s, i // pt], i % pt
                kq[d, h, :, j], ks[d, h, j], vq[d, h, :, j], vs[d, h, :, j] = kq[p, h, :, b2], ks[p, h, b2], vq[p, h, :, b2], vs[p, h, :, b2]
                want_w[s, h, i] = w[s, h, kept[s, h, i]]
    got = dev.numpy()
    for name in ("kq", "vq"):
        assert np.array_equal(got[name], arrays[name]), name
    for name in ("ks", "vs"):
        assert np.array_equal(got[name].view(np.uint8), arrays[name]), name
    assert np.array_equal(w_out.cpu().numpy(), want_w)


def test_choice_and_move_from_a_graph(yahkv, torch_gpu):
    torch = torch_gpu
    rng = np.random.default_rng(1)
    lens, budget, pt = [400, 33, 200], 100, 32
    g = yahkv.geometry(8, 8, 2, 128, pt, 64)
    b = yahkv.pool_bytes(g)
    dev, ref = yahkv.DevicePools(g), yahkv.DevicePools(g)
    arrays = {k: rng.integers(0, 256, b[k], dtype=np.uint8) for k in b}
    perm = rng.permutation(64).astype(np.int32)
    t = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()
    table, dst = t(perm[:39].reshape(3, 13)), t(perm[39:51].reshape(3, 4))
    seq_len, w = t(np.array(lens, np.int32)), torch.rand(3, 2, 400, device="cuda")
    kept, n_kept = torch.zeros(3, 2, budget, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    w_out = torch.zeros(3, 2, budget, device="cuda")

    def run(pools, kept, n_kept, w_out):
        yahkv.evict_select(g, seq_len, 400, w, budget, 4, 16, kept=kept, n_kept=n_kept)
        yahkv.evict_compact(pools, table, kept, n_kept, dst, w, w_out)

    dev.load(arrays)
    run(dev, kept, n_kept, w_out)
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            run(dev, kept, n_kept, w_out)
    for i in range(3):
        w.copy_(torch.rand(3, 2, 400, device="cuda"))
        seq_len.copy_(t(np.array([lens[(i + j) % 3] for j in range(3)], np.int32)))
        want = [torch.zeros_like(x) for x in (kept, n_kept, w_out)]
        dev.load(arrays), ref.load(arrays)
        run(ref, *want)
        w_out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip((kept, n_kept, w_out, dev.kq, dev.ks, dev.vq, dev.vs), (*want, ref.kq, ref.ks, ref.vq, ref.vs)):
            assert torch.equal(x, y), i


def test_compact_clamps_what_it_reads(yahkv, torch_gpu):
    """Kept positions past the table and page numbers past the pool are cut to them, a count past the budget to the budget."""
    torch = torch_gpu
    g = yahkv.geometry(8, 8, 2, 128, 16, 4)
    dev = yahkv.DevicePools(g, fill=3)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    kept = t([[[0, 5, 2 ** 31 - 1, -1]] * 2])
    w, w_out = torch.rand(1, 2, 20, device="cuda"), torch.zeros(1, 2, 4, device="cuda")
    yahkv.evict_compact(dev, t([[0, 10 ** 9]]), kept, t([99]), t([[-5]]), w, w_out)
    torch.cuda.synchronize()
    assert torch.equal(w_out[0], w[0][:, [0, 5, 19, 0]]) and bool((dev.kq == 3).all())


def test_fork_answer_evict_continue(yahkv, torch_gpu):
    """A document appended once with scaled rotary positions, three forks that answer it in shared steps while their keys are
    weighed, a cut of every fork to a budget into fresh pages, and further steps at positions that no longer are cache slots:
    attention after the cut equals the closed form over exactly the kept keys and those that came after."""
    torch = torch_gpu
    n_q, n_kv, hd, pt, doc, budget, sink, recent, scale = 8, 2, 128, 16, 200, 96, 2, 16, 128 ** -0.5
    n, steps_before, steps_after = 3, 4, 3
    total = doc + steps_before
    P = 64
    g = yahkv.geometry(8, n_q, n_kv, hd, pt, P)
    og = oracle.geometry(8, n_q, n_kv, hd, pt, P)
    dev, pool = yahkv.DevicePools(g), yahkv.PagePool(P)
    pool.shuffle(5)
    t = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(9)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(torch.bfloat16)
    r = yahkv.Rotary(hd, 1e6, scaling="yarn", factor=4.0, original_len=128.0, normalise=True)
    full = doc // pt
    common = pool.alloc(full + (doc % pt > 0))
    yahkv.rotary_append(dev, t([common]), t([0]), r, rnd(1, doc, n_kv, hd), rnd(1, doc, n_kv, hd))
    width = (total + steps_after + pt - 1) // pt
    rows, shared = [], common[:full]
    for i in range(n):                                                  # forks share the full pages, the last one is copied
        if i:
            pool.retain(shared)
        own = pool.alloc(width - full)
        yahkv.copy_pages(dev, t([common[full]]), t([own[0]]))
        rows.append(shared + own)
    pool.free([common[full]])                                           # (every fork has its own copy of it)
    table = t(rows)
    weights = torch.zeros(n, n_kv, width * pt, device="cuda")
    first, sh = t([0, n]), t([doc])
    for step in range(steps_before):
        at = t([doc + step] * n)
        x = rnd(n, 1, n_q + 2 * n_kv, hd)
        q = yahkv.rotary_append(dev, table, at, r, x[:, :, n_q:n_q + n_kv], x[:, :, n_q + n_kv:], x[:, :, :n_q], q_out_dtype=torch.float16)
        q = q.view(n, n_q, hd)
        a = yahkv.decode_attend_shared(dev, table, at + 1, first, sh, doc, doc % 64 + step + 1, q, scale)
        b = yahkv.decode_attend_weights(dev, table, at + 1, doc + step + 1, q, scale, weights, weights_in=weights)
        check(torch, a, b.double().cpu().numpy(), torch.float32)
    assert torch.allclose(weights.sum(-1), torch.full((n, n_kv), steps_before * n_q / n_kv, device="cuda"), rtol=1e-4)
    lens = t([total] * n)
    kept, n_kept = yahkv.evict_select(g, lens, total, weights, budget, sink, recent)
    fresh = [pool.alloc((budget + steps_after + pt - 1) // pt) for _ in range(n)]
    slim = torch.zeros(n, n_kv, len(fresh[0]) * pt, device="cuda")
    yahkv.evict_compact(dev, table, kept, n_kept, t(fresh), weights, slim)
    before = {k: v.copy() for k, v in dev.numpy().items()}
    for row in rows:
        pool.free(row)
    host = oracle.HostPools(og)
    for name, arr in host.arrays().items():
        arr.reshape(-1)[:] = before[name].reshape(-1)
    new_table, G = t(fresh), n_q // n_kv
    keys, values = [], []
    for i in range(n):                                                  # the kept keys, read through the old tables
        (ks, kc), (vs, vc) = logical_blocks(host.arrays(), og, np.array(rows[i]), total)
        k, v = dequant(ks, kc), dequant(vs, vc)
        idx = kept[i].cpu().numpy()
        keys.append(np.stack([k[idx[h], h] for h in range(n_kv)], 1)), values.append(np.stack([v[idx[h], h] for h in range(n_kv)], 1))
    for step in range(steps_after):
        slot, pos = n_kept + step, t([[total + step]] * n)
        x = rnd(n, 1, n_q + 2 * n_kv, hd)
        q = yahkv.rotary_append(dev, new_table, slot, r, x[:, :, n_q:n_q + n_kv], x[:, :, n_q + n_kv:], x[:, :, :n_q], positions=pos,
                                q_out_dtype=torch.float16).view(n, n_q, hd)
        out = yahkv.decode_attend_weights(dev, new_table, slot + 1, budget + step + 1, q, scale, slim, weights_in=slim)
        for name, arr in host.arrays().items():
            arr.reshape(-1)[:] = dev.numpy()[name].reshape(-1)
        for i in range(n):
            (ks, kc), (vs, vc) = logical_blocks(host.arrays(), og, np.array(fresh[i]), budget + step + 1)
            k, v = dequant(ks, kc), dequant(vs, vc)
            assert np.array_equal(k[:budget], keys[i][:budget]) and np.array_equal(v[:budget], values[i][:budget])
            for hq in range(n_q):
                s = k[:, hq // G].astype(np.float64) @ q[i, hq].double().cpu().numpy() * scale
                p = np.exp(s - s.max())
                want = (p / p.sum()) @ v[:, hq // G].astype(np.float64)
                assert np.abs(out[i, hq].double().cpu().numpy() - want).max() <= 2e-3 * np.abs(want).max()
    assert pool.free_count == P - sum(len(f) for f in fresh)
