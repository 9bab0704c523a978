"""Decode attention over shared prefixes (yahkv_decode_attend_shared) against the closed form in float64, and against the
plain decode attention on the same tables.

Tolerance: the library's 2e-3 of the largest value (K, V and the softmax numerators enter the matrix unit as f16, half a step
2^-11 each, over sums of independent terms); a 16-bit output adds half a step of its own value, finfo.eps / 2."""
import numpy as np
import pytest

import oracle
from helpers import to_bf16_f32
from test_gpu_decode import closed

pytestmark = pytest.mark.gpu
TOL = 2e-3


def batch(yahkv, torch, fmt, n_q, n_kv, hd, pt, groups, seed, fill=0x7F, spare=2):
    """groups: [(shared_len, [lengths])]. Full pages of a prefix are shared, the rest is every sequence's own."""
    rng = np.random.default_rng(seed)
    lens = [n for _, ls in groups for n in ls]
    pages_of = lambda n: (n + pt - 1) // pt
    total = sum(sh // pt + sum(max(pages_of(n) - sh // pt, 0) for n in ls) for sh, ls in groups)
    # a sequence shorter than its prefix keeps the row of the shared pages
    g = oracle.geometry(fmt, n_q, n_kv, hd, pt, total + spare)
    perm, at = rng.permutation(g.n_pages).astype(np.int32), 0
    table = np.zeros((len(lens), max(max(pages_of(max(n, sh)) for sh, ls in groups for n in ls), 1)), np.int32)
    host = oracle.HostPools(g, fill=fill)
    s = 0
    rows = lambda n: to_bf16_f32(rng.standard_normal((1, n, n_kv, hd)))
    for sh, ls in groups:
        common, at = perm[at:at + sh // pt], at + sh // pt
        pk, pv = rows(sh) if sh else None, rows(sh) if sh else None
        for n in ls:
            table[s, :len(common)] = common
            own = max(pages_of(n) - len(common), 0)
            table[s, len(common):len(common) + own] = perm[at:at + own]
            at += own
            if n:
                k, v = rows(n), rows(n)
                m = min(sh, n)
                if m:
                    k[:, :m], v[:, :m] = pk[:, :m], pv[:, :m]
                oracle.append(host, table[s:s + 1], [0], None, k, v)
            s += 1
        if sh // pt:  # the prefix's pages are whole even where no sequence reaches their end
            oracle.append(host, table[s - 1:s], [0], None, pk[:, :sh // pt * pt], pv[:, :sh // pt * pt])
    dev = yahkv.DevicePools(yahkv.geometry(fmt, n_q, n_kv, hd, pt, g.n_pages))
    dev.load(host.arrays())
    first = np.cumsum([0] + [len(ls) for _, ls in groups])
    t = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")
    shared = [sh for sh, _ in groups]
    tail = max([1] + [n - (sh // 64 * 64 if n >= sh // 64 * 64 else 0) for sh, ls in groups for n in ls])
    q = torch.from_numpy(rng.standard_normal((len(lens), n_q, hd)).astype(np.float32)).cuda()
    return g, table, host, dev, lens, q, dict(table=t(table), seq_len=t(lens), group_first=t(first), shared_len=t(shared),
                                              max_shared_len=max(shared), max_tail_len=tail)


def check(torch, got, want, dtype):
    got = got.double().cpu().numpy()
    half = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    assert np.all(np.isfinite(got))
    err = np.abs(got - want)
    assert np.all(err <= TOL * np.abs(want).max() + half * 1.002 * np.abs(want)), float(err.max() / np.abs(want).max())


HEADS = [(24, 4, 256), (32, 8, 128), (8, 8, 128), (8, 1, 256), (3, 1, 128)]


@pytest.mark.parametrize("fmt,pt", [(8, 64), (8, 16), (4, 32), (4, 64)])
@pytest.mark.parametrize("n_q,n_kv,hd", HEADS)
def test_one_prefix(yahkv, torch_gpu, n_q, n_kv, hd, fmt, pt):
    torch = torch_gpu
    g, table, host, dev, lens, q, a = batch(yahkv, torch, fmt, n_q, n_kv, hd, pt, [(300, [300, 301, 420, 364, 999])], fmt * pt + hd)
    scale = hd ** -0.5
    for kind, dtype in ((torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32)):
        x = q.to(kind)
        want = closed(g, table, host, lens, x.double().cpu().numpy(), scale)
        check(torch, yahkv.decode_attend_shared(dev, q=x, scale=scale, out_dtype=dtype, **a), want, dtype)


@pytest.mark.parametrize("groups", [
    [(0, [1])], [(0, [0, 5, 64, 65])], [(63, [63, 64, 200])], [(64, [64, 64, 65])], [(65, [65, 65])], [(128, [128])],
    [(129, [0, 1, 63, 64, 127, 128, 129, 400])],                                     # some shorter than the prefix, one empty
    [(1000, [0, 0, 0])],                                                             # nothing but empty ones
    [(200, [200, 264]), (0, [77]), (640, [700] * 9), (64, [10, 64, 3])],             # groups side by side, one without a prefix
    [(192, [250 + i for i in range(23)])], [(3000, [3000 + i for i in range(45)])],  # more rows than a workgroup's
    [(64 * i + 64, [64 * i + 70]) for i in range(9)]])                               # every sequence a group of its own
def test_lengths_and_groups(yahkv, torch_gpu, groups):
    torch = torch_gpu
    n_q, n_kv, hd, pt = 12, 2, 128, 32
    g, table, host, dev, lens, q, a = batch(yahkv, torch, 8, n_q, n_kv, hd, pt, groups, len(groups) + groups[0][0])
    gate = torch.randn(len(lens), n_q, hd, device="cuda")
    want = closed(g, table, host, lens, q.half().double().cpu().numpy(), 0.1, gate.double().cpu().numpy())
    got = yahkv.decode_attend_shared(dev, q=q.half(), scale=0.1, gate=gate, **a)
    check(torch, got, want, torch.float32)
    for s, n in enumerate(lens):
        assert n > 0 or not got[s].any()
    if max(lens) == 0:
        return
    plain = yahkv.decode_attend(dev, a["table"], a["seq_len"], max(lens), q.half(), 0.1, gate=gate)
    check(torch, got, plain.double().cpu().numpy(), torch.float32)
    # larger host bounds than needed change nothing but the sums' order
    a.update(max_shared_len=a["max_shared_len"] + 5000, max_tail_len=a["max_tail_len"] + 777)
    check(torch, yahkv.decode_attend_shared(dev, q=q.half(), scale=0.1, gate=gate, **a), want, torch.float32)


@pytest.mark.parametrize("fmt,pt", [(8, 64), (8, 32), (8, 16), (4, 64), (4, 32), (4, 16)])
@pytest.mark.parametrize("n_q,n_kv,hd", [(24, 4, 256), (32, 8, 128), (8, 1, 256), (5, 1, 128)])
def test_bounds_of_a_large_call(yahkv, torch_gpu, n_q, n_kv, hd, fmt, pt):
    """The host bounds of a long context choose as many row blocks a wave as registers hold, and tails in a launch of their
    own, whatever the lengths on the device are."""
    torch = torch_gpu
    groups = [(640, [650 + 7 * i for i in range(20)]), (0, [3]), (200, [100, 200, 330])]
    g, table, host, dev, lens, q, a = batch(yahkv, torch, fmt, n_q, n_kv, hd, pt, groups, fmt + pt + hd)
    a.update(max_shared_len=65536, max_tail_len=40000)
    want = closed(g, table, host, lens, q.half().double().cpu().numpy(), hd ** -0.5)
    check(torch, yahkv.decode_attend_shared(dev, q=q.half(), scale=hd ** -0.5, **a), want, torch.float32)


def test_more_groups_than_lanes(yahkv, torch_gpu):
    torch = torch_gpu
    groups = [(64 * (i % 4), [64 * (i % 4) + 1 + i] * (1 + i % 3)) for i in range(131)]
    g, table, host, dev, lens, q, a = batch(yahkv, torch, 8, 4, 2, 128, 64, groups, 131)
    want = closed(g, table, host, lens, q.half().double().cpu().numpy(), 0.1)
    for bound in (192, 65536):
        a["max_shared_len"] = bound
        check(torch, yahkv.decode_attend_shared(dev, q=q.half(), scale=0.1, **a), want, torch.float32)


def test_bounds_clamp(yahkv, torch_gpu):
    """A prefix beyond max_shared_len counts as tail; a shared_len that is negative or past the table is cut to it."""
    torch = torch_gpu
    g, table, host, dev, lens, q, a = batch(yahkv, torch, 8, 8, 2, 128, 16, [(256, [256, 300, 280])], 5)
    want = closed(g, table, host, lens, q.half().double().cpu().numpy(), 0.1)
    b = dict(a, max_shared_len=128, max_tail_len=300 - 128)
    check(torch, yahkv.decode_attend_shared(dev, q=q.half(), scale=0.1, **b), want, torch.float32)
    b = dict(a, shared_len=torch.tensor([-7], dtype=torch.int32, device="cuda"), max_tail_len=300)
    check(torch, yahkv.decode_attend_shared(dev, q=q.half(), scale=0.1, **b), want, torch.float32)
    # the table reaches 19 pages of 16 tokens: 304, of which whole tiles 256
    b = dict(a, shared_len=torch.tensor([2 ** 31 - 1], dtype=torch.int32, device="cuda"), max_shared_len=2 ** 31 - 1 - 64)
    check(torch, yahkv.decode_attend_shared(dev, q=q.half(), scale=0.1, **b), want, torch.float32)


def test_large_values_stay_finite(yahkv, torch_gpu):
    """Blocks of values up to the largest f16 scale times 127: the products saturate instead of becoming infinite."""
    torch = torch_gpu
    g = yahkv.geometry(8, 8, 1, 128, 64, 3)
    dev = yahkv.DevicePools(g, fill=1)
    dev.vs.view(torch.float16).fill_(60000.0)
    dev.ks.view(torch.float16).fill_(2.0)
    dev.vq.view(torch.int8).fill_(127)
    t = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    q = torch.randn(2, 8, 128, device="cuda").half()
    out = yahkv.decode_attend_shared(dev, torch.tensor([[0, 1], [0, 2]], dtype=torch.int32, device="cuda"), t(64, 64), t(0, 2), t(64),
                                     64, 64, q, 0.1)
    assert torch.all((out - 65504.0).abs() <= 65504.0 * TOL)


def test_non_finite_keys_stay_with_those_who_see_them(yahkv, torch_gpu):
    """A NaN scale behind every sequence's end, or in prefix keys that only the longer sequences have, leaves the others alone."""
    torch = torch_gpu
    g, table, host, dev, lens, q, a = batch(yahkv, torch, 8, 8, 2, 128, 64, [(192, [192, 100, 300, 0])], 6)
    want = closed(g, table, host, lens, q.half().double().cpu().numpy(), 0.1)
    nan = torch.tensor(float("nan"), device="cuda", dtype=torch.float16)
    vs, ks = dev.vs.view(torch.float16).view(-1, 2, 4, 64), dev.ks.view(torch.float16).view(-1, 2, 64, 4)
    vs[table[2, 4], :, :, 300 - 256:], ks[table[2, 4], :, 300 - 256:] = nan, nan      # behind the longest sequence's end
    got = yahkv.decode_attend_shared(dev, q=q.half(), scale=0.1, **a)
    check(torch, got, want, torch.float32)
    vs[table[0, 2], 0, 1, 5] = nan                                                    # key 133: not sequence 1's
    got = yahkv.decode_attend_shared(dev, q=q.half(), scale=0.1, **a)
    assert torch.isnan(got[[0, 2]][:, :4, 32:64]).all() and torch.isfinite(got[1]).all() and not got[3].any()
    check(torch, got[1], want[1], torch.float32)


def test_same_bits_twice_and_from_a_graph(yahkv, torch_gpu):
    torch = torch_gpu
    g, table, host, dev, lens, q, a = batch(yahkv, torch, 8, 24, 4, 256, 64, [(640, [700 + 9 * i for i in range(7)]), (64, [500, 64])], 8)
    x = q.to(torch.bfloat16)
    ws = torch.empty(yahkv.decode_shared_workspace_bytes(dev.geom, 9, 2, a["max_shared_len"], a["max_tail_len"]), dtype=torch.uint8, device="cuda")
    out = torch.empty(x.shape, device="cuda")
    step = lambda: yahkv.decode_attend_shared(dev, q=x, scale=0.0625, out=out, workspace=ws, **a)
    step()
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            step()
    for i in range(3):
        x.copy_(torch.randn(x.shape, device="cuda"))
        a["seq_len"].add_(i)                  # lengths live on the device (the new keys were never written: NaN, so bits are compared)
        ws.random_(0, 256)
        step()
        want = out.clone()
        out.fill_(float("nan"))
        ws.random_(0, 256)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int32), want.view(torch.int32)) and (i or torch.isfinite(out).all()), i
        a["seq_len"].sub_(i)


def test_two_graphs_on_one_workspace(yahkv, torch_gpu):
    """A shared step and a weighing step, captured apart on the same workspace and replayed in turn: what each gives alone."""
    torch = torch_gpu
    g, table, host, dev, lens, q, a = batch(yahkv, torch, 8, 24, 4, 256, 64, [(640, [650, 700, 900]), (0, [70])], 12)
    q = q.half()
    need = max(yahkv.decode_shared_workspace_bytes(dev.geom, 4, 2, a["max_shared_len"], a["max_tail_len"]),
               yahkv.decode_weights_workspace_bytes(dev.geom, 4, 900))
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    out, w = torch.empty(4, 24, 256, device="cuda"), torch.zeros(4, 4, 900, device="cuda")
    out2 = torch.empty_like(out)
    steps = [lambda: yahkv.decode_attend_shared(dev, q=q, scale=0.0625, out=out, workspace=ws, **a),
             lambda: yahkv.decode_attend_weights(dev, a["table"], a["seq_len"], 900, q, 0.0625, w, out=out2, workspace=ws)]
    for s in steps:
        s()
    want = out.clone(), w.clone(), out2.clone()
    graphs, stream = [torch.cuda.CUDAGraph() for _ in steps], torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for graph, s in zip(graphs, steps):
            with torch.cuda.graph(graph, stream=stream):
                s()
    for i in range(3):
        for x in (out, w, out2):
            x.fill_(-1.0)
        torch.cuda.synchronize()
        for graph in (graphs if i % 2 else graphs[::-1]):
            graph.replay()
        torch.cuda.synchronize()
        for s, n in enumerate(lens):
            assert torch.equal(w[s, :, :n], want[1][s, :, :n])
        assert torch.equal(out, want[0]) and torch.equal(out2, want[2]), i


def test_workspace_too_small_is_refused(yahkv, torch_gpu):
    torch = torch_gpu
    g, table, host, dev, lens, q, a = batch(yahkv, torch, 8, 8, 2, 128, 16, [(64, [70])], 9)
    with pytest.raises(yahkv.YahkvError) as e:
        yahkv.decode_attend_shared(dev, q=q, scale=0.1, workspace=torch.empty(64, dtype=torch.uint8, device="cuda"), **a)
    assert e.value.status == -4


@pytest.mark.parametrize("fmt,n_q,n_kv,hd,pt,big", [(8, 24, 4, 256, 64, 60000.0), (8, 8, 2, 128, 16, 600.0), (8, 32, 8, 128, 32, 65504.0),
                                                    (4, 24, 4, 256, 32, 60000.0), (4, 8, 2, 128, 64, 9000.0)])
@pytest.mark.parametrize("bound", [0, 65536])
def test_keys_beyond_the_f16_range(yahkv, torch_gpu, fmt, n_q, n_kv, hd, pt, big, bound):
    """Keys whose values d * code are far beyond 65504, in prefixes and tails, next to ordinary ones: their scores are the plain
    decode attention's. The softmax scale brings the large ones' scores to a standard deviation of about four."""
    torch = torch_gpu
    groups = [(192, [192, 250, 300, 0]), (0, [70]), (640, [700] * 30)]
    g, table, host, dev, lens, q, a = batch(yahkv, torch, fmt, n_q, n_kv, hd, pt, groups, int(big) + hd)
    ks = dev.ks.view(torch.float16).view(-1, n_kv, pt, hd // 32)
    gen = torch.Generator(device="cuda").manual_seed(1)
    some = torch.rand(ks.shape[:3], generator=gen, device="cuda") < 0.3
    blocks = torch.rand(ks.shape, generator=gen, device="cuda")
    large = ((0.5 + 0.5 * blocks) * big).half()
    ks.copy_(torch.where(some[..., None] & (blocks > 0.25) & torch.isfinite(ks), large, ks))
    for name, arr in host.arrays().items():
        arr.reshape(-1)[:] = dev.numpy()[name].reshape(-1)
    rms = {8: 45.0, 4: 3.0}[fmt] * 0.75 * big                          # of a large key's values
    scale = 4.0 / (rms * hd ** 0.5)
    if bound:
        a.update(max_shared_len=bound, max_tail_len=40000)
    want = closed(g, table, host, lens, q.half().double().cpu().numpy(), scale)
    plain = yahkv.decode_attend(dev, a["table"], a["seq_len"], max(lens), q.half(), scale)
    check(torch, plain, want, torch.float32)
    check(torch, yahkv.decode_attend_shared(dev, q=q.half(), scale=scale, **a), want, torch.float32)


@pytest.mark.parametrize("fmt,hd,pt", [(8, 256, 64), (8, 128, 16), (4, 128, 64), (4, 256, 32)])
@pytest.mark.parametrize("large", ["ks", "vs", "both"])
def test_nan_and_infinite_queries_give_nan_beside_large_scales(yahkv, torch_gpu, fmt, hd, pt, large):
    """What a query's own values make of its row does not depend on the magnitude of the keys and values it meets."""
    torch = torch_gpu
    groups = [(192, [192, 250, 300]), (0, [70])]
    g, table, host, dev, lens, q, a = batch(yahkv, torch, fmt, 8, 2, hd, pt, groups, hd + pt)
    for name in ("ks", "vs"):
        if large in (name, "both"):
            s = getattr(dev, name).view(torch.float16)
            s.copy_(torch.where(torch.isfinite(s), torch.full_like(s, 60000.0), s))
    q = q.half()
    bad = {(0, 3): float("nan"), (2, 5): float("inf"), (3, 0): float("nan")}
    for (s, h), v in bad.items():
        q[s, h, 7 * h + 1] = v
    out = yahkv.decode_attend_shared(dev, q=q, scale=1e-7, **a)
    for s in range(4):
        for h in range(8):
            assert (torch.isnan(out[s, h]) if (s, h) in bad else torch.isfinite(out[s, h])).all(), (s, h)


@pytest.mark.parametrize("leaders", [[0], [100], [0, 63, 191], [0] * 70, [5, 0] * 40])
@pytest.mark.parametrize("bound", [0, 65536])
def test_a_group_led_by_sequences_shorter_than_its_prefix(yahkv, torch_gpu, leaders, bound):
    """Sequences that are shorter than the prefix's tiles (idle slots among them) are read through their own rows alone, also at
    the head of a group: their rows name other pages than the prefix's."""
    torch = torch_gpu
    n_q, n_kv, hd, pt = 8, 2, 128, 32
    groups = [(192, leaders + [250, 0, 300]), (0, [70]), (130, [5, 128, 200]), (256, [0, 9])]
    g, table, host, dev, lens, q, a = batch(yahkv, torch, 8, n_q, n_kv, hd, pt, groups, len(leaders) + sum(leaders), spare=4 * len(leaders) + 16)
    rng = np.random.default_rng(3)
    free = [p for p in range(g.n_pages) if p not in set(table.reshape(-1).tolist())]
    at, n = 0, len(leaders)
    for s in list(range(n)) + [n + 1, n + 4, len(lens) - 2, len(lens) - 1]:
        need = max((lens[s] + pt - 1) // pt, 1)
        table[s] = free[at]                                                # a page that holds nothing written
        table[s, :need] = free[at:at + need]
        at += need
        if lens[s]:
            oracle.append(host, table[s:s + 1], [0], None, *(to_bf16_f32(rng.standard_normal((1, lens[s], n_kv, hd))) for _ in range(2)))
    dev.load(host.arrays())
    a["table"] = torch.from_numpy(table).cuda()
    if bound:
        a.update(max_shared_len=bound, max_tail_len=40000)
    want = closed(g, table, host, lens, q.half().double().cpu().numpy(), 0.1)
    got = yahkv.decode_attend_shared(dev, q=q.half(), scale=0.1, **a)
    check(torch, got, want, torch.float32)
    for s, m in enumerate(lens):
        assert m > 0 or not got[s].any()


@pytest.mark.parametrize("fmt,n_q,n_kv,hd,pt", [(8, 24, 4, 256, 64), (8, 8, 2, 128, 16), (4, 32, 8, 128, 32), (4, 24, 4, 256, 64)])
@pytest.mark.parametrize("bound", [0, 65536])
@pytest.mark.parametrize("kind", ["keys", "keys next to ordinary ones", "scale", "no scale"])
def test_scores_far_from_zero(yahkv, torch_gpu, fmt, n_q, n_kv, hd, pt, bound, kind):
    """Scores of 1e9 and 1e31, where a unit of their last place is far more than one (a softmax of them is its largest score's
    key), and scores that are all next to nothing (a mean). Large keys are powers of two times their codes, so that they are
    exact in f16 and the largest score is too."""
    torch = torch_gpu
    groups = [(192, [192, 250, 300, 0]), (0, [70, 1]), (640, [700] * 30)]
    g, table, host, dev, lens, q, a = batch(yahkv, torch, fmt, n_q, n_kv, hd, pt, groups, hd + pt, fill=0x7F if kind == "keys" else 0x11)
    scale = {"scale": 1e30, "no scale": 1e-38}.get(kind, hd ** -0.5)
    if kind.startswith("keys"):
        ks = dev.ks.view(torch.float16).view(-1, n_kv, pt, hd // 32)
        gen = torch.Generator(device="cuda").manual_seed(1)
        some = torch.rand(ks.shape[:3], generator=gen, device="cuda") < (2.0 if kind == "keys" else 0.1)
        ks.copy_(torch.where(some[..., None] & torch.isfinite(ks), torch.full_like(ks, 32768.0), ks))
        for name, arr in host.arrays().items():
            arr.reshape(-1)[:] = dev.numpy()[name].reshape(-1)
        q *= 200.0
    if bound:
        a.update(max_shared_len=bound, max_tail_len=40000)
    want = closed(g, table, host, lens, q.half().double().cpu().numpy(), scale)
    check(torch, yahkv.decode_attend_shared(dev, q=q.half(), scale=scale, **a), want, torch.float32)


@pytest.mark.parametrize("fmt,n_q,n_kv,hd,pt", [(8, 24, 4, 256, 64), (8, 8, 2, 128, 16), (4, 32, 8, 128, 32), (4, 24, 4, 256, 64)])
def test_unwritten_slots_have_no_say(yahkv, torch_gpu, fmt, n_q, n_kv, hd, pt):
    """The same bits whatever the slots behind every sequence's end hold: zeros, ordinary codes and scales, NaN, large scales. (The
    written keys are small ones, whose scales do not survive a factor of 2^-7 in f16.)"""
    torch = torch_gpu
    got = []
    for fill in (0x00, 0x21, 0x7F, 0xFF, 0x7B):
        g, table, host, dev, lens, q, a = batch(yahkv, torch, fmt, n_q, n_kv, hd, pt, [(192, [192, 250, 300, 0]), (0, [70, 1]), (640, [700, 641])],
                                                hd, fill=fill)
        dev.ks.view(torch.float16).mul_(0.01)
        got.append(yahkv.decode_attend_shared(dev, q=(q * 100).half(), scale=hd ** -0.5, **a))
    for x in got[1:]:
        assert torch.equal(x, got[0])
