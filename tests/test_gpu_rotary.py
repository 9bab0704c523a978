"""Rotary positions on the GPU (yahkv_rotary_apply, yahkv_rotary_append) against the definition in float64.

Tolerance of an f32 result, in u = 2^-24 of the larger of the row's magnitudes: the sum of up to 512 squares 8 + 6 steps,
division, root and reciprocal 3, two products 2: 19, halved for the sum by the root, so 12 u on a normalised value; cosine and
sine 4 u (two units of the last place at most), the remainder's rounding pi / 4 u, the magnitude u; a product and a sum 2 u: 20 u
on each of two terms, 40 u = 2.4e-6 of (|x| + |y|) at most, taken as 2.4e-6 of twice the row's largest value times the
magnitude. A 16-bit result adds half a step of its own value, finfo.eps / 2."""
import math

import numpy as np
import pytest

import oracle
from helpers import make_tables
from test_host_serving import exact_turns, frequencies

pytestmark = pytest.mark.gpu
SPEC = dict(none=0, linear=1, ntk=2, yarn=3, bands=4)


def want_rows(x, pos, dim, layout, scaling, first=0, weight=None, eps=1e-6, normalise=False, theta=1e4):
    """x float64 [n][t][heads][D], pos [n][t]."""
    low, high = (1.0, 4.0) if scaling == "bands" else (1.0, 32.0)
    f = frequencies(dim, SPEC[scaling], theta, 8.0, 4096.0, low, high)
    mag = 0.1 * math.log(8.0) + 1 if scaling == "yarn" else 1.0
    # angles of far positions in extended precision
    a = (np.asarray(pos, np.longdouble)[..., None, None] * f.astype(np.longdouble)) % np.longdouble("6.28318530717958647692528676655900577")
    c, s = np.cos(a).astype(np.float64) * mag, np.sin(a).astype(np.float64) * mag
    x = np.array(x, np.float64)
    if normalise:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        if weight is not None:
            x = x * weight
    out = x.copy()
    i0 = first + (np.arange(dim // 2) if layout == "half" else 2 * np.arange(dim // 2))
    i1 = i0 + (dim // 2 if layout == "half" else 1)
    out[..., i0] = x[..., i0] * c - x[..., i1] * s
    out[..., i1] = x[..., i1] * c + x[..., i0] * s
    return out


def close(torch, got, want, dtype):
    got = got.double().cpu().numpy()
    half = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    tiny = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}[dtype]        # half a subnormal step
    tol = 2.4e-6 * 2 * 1.3 * np.abs(want).max(-1, keepdims=True) + half * np.abs(want) * 1.001 + tiny
    assert got.shape == want.shape and np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / tol).max())


def make(yahkv, dim, layout, scaling, **kw):
    low, high = (1.0, 4.0) if scaling == "bands" else (1.0, 32.0)
    return yahkv.Rotary(dim, kw.pop("theta", 1e4), layout=layout, scaling=scaling, factor=8.0, original_len=4096.0, low=low, high=high, **kw)


@pytest.mark.parametrize("scaling", sorted(SPEC))
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_scalings_and_far_positions(yahkv, torch_gpu, layout, scaling):
    torch = torch_gpu
    gen = torch.Generator(device="cuda").manual_seed(1)
    pos = np.array([[0], [1], [-1], [4095], [123456], [2 ** 31 - 1], [-2 ** 31], [1000003]])
    q = torch.randn(8, 1, 3, 128, generator=gen, device="cuda")
    k = torch.randn(8, 1, 1, 128, generator=gen, device="cuda")
    r = make(yahkv, 128, layout, scaling)
    qo, ko = yahkv.rotary_rows(r, torch.tensor(pos, dtype=torch.int32, device="cuda"), q, k)
    # the frequencies are doubles on both sides, rounded apart: up to 2^-46 relative (tested on the host), which at position
    # 2^31 is 3e-5 radians; nearer positions show it less
    spread = np.abs(pos)[..., None, None] * 64 * 2.0 ** -53
    for got, x in ((qo, q), (ko, k)):
        want = want_rows(x.cpu().numpy(), pos, 128, layout, scaling)
        tol = (2.4e-6 * 2.6 + 2.6 * spread) * np.abs(want).max(-1, keepdims=True)
        assert np.all(np.abs(got.double().cpu().numpy() - want) <= tol)


@pytest.mark.parametrize("scaling", sorted(SPEC))
@pytest.mark.parametrize("theta", [1e4, 1e7])
def test_angles_of_far_positions(yahkv, torch_gpu, theta, scaling):
    """Pairs (1, 0) become the cosine and sine themselves: against frequencies of 60 digits, so that a far position shows what the
    table lacks. Tolerance: 4 u = 2.4e-7 of a sine (above), and of the angle 2^-63 turns times the position (the table, tested on
    the host) and 2^-32 turns (the bits of the fraction that the sine drops): 2^-32 + 2^-32 turns, 2.9e-9 radians."""
    from fractions import Fraction
    torch = torch_gpu
    pos = [0, 1, -1, 4095, 123456, 10 ** 6 + 3, 2 ** 28 + 1, 2 ** 31 - 1, -2 ** 31, -2 ** 31 + 12345]
    low, high = (1.0, 4.0) if scaling == "bands" else (1.0, 32.0)
    f = [Fraction(x) for x in exact_turns(64, SPEC[scaling], theta, 8.0, 4096.0, low, high)]
    a = np.array([[float(p * x % 1) for x in f] for p in pos]) * 2 * np.pi
    q = torch.zeros(len(pos), 1, 1, 64, device="cuda")
    q[..., :32] = 1.0
    r = make(yahkv, 64, "half", scaling, theta=theta, magnitude=1.0)
    y, _ = yahkv.rotary_rows(r, torch.tensor(pos, dtype=torch.int32, device="cuda")[:, None], q)
    y = y.double().cpu().numpy()[:, 0, 0]
    assert np.abs(y[:, :32] - np.cos(a)).max() <= 2.4e-7 + 2.9e-9 and np.abs(y[:, 32:] - np.sin(a)).max() <= 2.4e-7 + 2.9e-9


@pytest.mark.parametrize("d,dim,first", [(8, 8, 0), (40, 16, 8), (64, 32, 32), (80, 80, 0), (96, 64, 4), (128, 128, 0), (192, 64, 128),
                                         (256, 64, 0), (256, 256, 0), (512, 512, 0), (512, 128, 100)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_part_of_the_head_and_types(yahkv, torch_gpu, layout, d, dim, first):
    torch = torch_gpu
    gen = torch.Generator(device="cuda").manual_seed(d + dim)
    pos = torch.randint(0, 5000, (2, 3), generator=gen, device="cuda", dtype=torch.int32)
    w = 1 + 0.3 * torch.randn(d, generator=gen, device="cuda")
    for n, (src, dst) in enumerate(((torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float32, torch.float16))):
        q = torch.randn(2, 3, 5, d, generator=gen, device="cuda").to(src)
        k = torch.randn(2, 3, 2, d, generator=gen, device="cuda").to(src)
        r = make(yahkv, dim, layout, "none", first_dim=first, normalise=n != 1, q_weight=w if n == 0 else None, k_weight=w)
        qo, ko = yahkv.rotary_rows(r, pos, q, k, out_dtype=dst)
        p = pos.cpu().numpy()
        w64 = w.double().cpu().numpy()
        close(torch, qo, want_rows(q.double().cpu().numpy(), p, dim, layout, "none", first, w64 if n == 0 else None, normalise=n != 1), dst)
        close(torch, ko, want_rows(k.double().cpu().numpy(), p, dim, layout, "none", first, w64, normalise=n != 1), dst)


@pytest.mark.parametrize("n,new", [(1, 1), (3, 1), (1, 1100), (2, 5)])
def test_strided_in_place_and_alone(yahkv, torch_gpu, n, new):
    """Slices of one fused projection, a head-major tensor, rotation in place, k without q; the rest of the buffer untouched."""
    torch = torch_gpu
    gen = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(n, new, 12, 128, generator=gen, device="cuda").to(torch.bfloat16)
    before = x.clone()
    pos = torch.randint(0, 300000, (n, new), generator=gen, device="cuda", dtype=torch.int32)
    r = make(yahkv, 64, "half", "linear", normalise=True)
    q, k = x[:, :, :8], x[:, :, 8:10]
    want_q = want_rows(before[:, :, :8].double().cpu().numpy(), pos.cpu().numpy(), 64, "half", "linear", normalise=True)
    want_k = want_rows(before[:, :, 8:10].double().cpu().numpy(), pos.cpu().numpy(), 64, "half", "linear", normalise=True)
    qo, ko = yahkv.rotary_rows(r, pos, q, k)                                  # out of place: strided in, dense out
    close(torch, qo, want_q, torch.bfloat16)
    close(torch, ko, want_k, torch.bfloat16)
    head_major = torch.zeros(n, 8, new, 128, device="cuda", dtype=torch.bfloat16).transpose(1, 2)
    yahkv.rotary_rows(r, pos, q, q_out=head_major)
    assert torch.equal(head_major, qo)
    only = yahkv.rotary_rows(r, pos, k=k)
    assert only[0] is None and torch.equal(only[1], ko)
    assert torch.equal(x, before)
    yahkv.rotary_rows(r, pos, q, k, q_out=q, k_out=k)                         # in place
    assert torch.equal(x[:, :, :8], qo) and torch.equal(x[:, :, 8:10], ko) and torch.equal(x[:, :, 10:], before[:, :, 10:])


@pytest.mark.parametrize("tokens", [2, 1030])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_many_rows_a_token_in_place(yahkv, torch_gpu, tokens, layout):
    """More rows than a workgroup has on its way at once, an odd number of them."""
    torch = torch_gpu
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    x = torch.randn(1, tokens, 40, 256, generator=gen, device="cuda")
    pos = torch.randint(-5, 100000, (1, tokens), generator=gen, device="cuda", dtype=torch.int32)
    r = make(yahkv, 128, layout, "ntk", first_dim=64)
    want = want_rows(x.double().cpu().numpy(), pos.cpu().numpy(), 128, layout, "ntk", first=64)
    yahkv.rotary_rows(r, pos, x[:, :, :37], x[:, :, 37:], q_out=x[:, :, :37], k_out=x[:, :, 37:])
    close(torch, x, want, torch.float32)


def test_repeated_source_rows(yahkv, torch_gpu):
    """One row for all heads and all sequences (strides of 0) on the way in; on the way out it is refused."""
    torch = torch_gpu
    x = torch.randn(1, 5, 1, 128, device="cuda").half()
    r = make(yahkv, 64, "half", "none")
    pos = torch.arange(15, dtype=torch.int32, device="cuda").view(3, 5)
    got, _ = yahkv.rotary_rows(r, pos, x.expand(3, 5, 4, 128))
    want, _ = yahkv.rotary_rows(r, pos, x.expand(3, 5, 4, 128).contiguous())
    assert torch.equal(got, want)
    with pytest.raises(yahkv.YahkvError):
        yahkv.rotary_rows(r, pos, x.expand(3, 5, 4, 128), q_out=torch.empty_like(x).expand(3, 5, 4, 128))


def test_untouched_dims_pass_through_infinities(yahkv, torch_gpu):
    """Dims that are not rotated are the source's bits, NaN and infinities among them; a pair with one is not finite."""
    torch = torch_gpu
    x = torch.randn(1, 1, 2, 64, device="cuda")
    x[0, 0, 0, 40], x[0, 0, 1, 63], x[0, 0, 1, 0] = float("inf"), float("nan"), float("inf")
    y, _ = yahkv.rotary_rows(make(yahkv, 32, "half", "none"), torch.tensor([[5]], dtype=torch.int32, device="cuda"), x)
    assert torch.equal(y[..., 32:].view(torch.int32), x[..., 32:].view(torch.int32))
    assert torch.isfinite(y[0, 0, 0, :32]).all() and not torch.isfinite(y[0, 0, 1, [0, 16]]).any()


def append_case(yahkv, torch, fmt, n_q, n_kv, hd, pt, starts, new, layout, dim, first, src, seed, n_valid=None, far=0):
    rng = np.random.default_rng(seed)
    pages = [(s + new + pt - 1) // pt for s in starts]
    g = oracle.geometry(fmt, n_q, n_kv, hd, pt, sum(pages) + 1)
    table = make_tables(rng, pages, g.n_pages)
    n = len(starts)
    x = torch.from_numpy(rng.standard_normal((n, new, n_q + 2 * n_kv, hd)).astype(np.float32)).cuda().to(src)
    dev = yahkv.DevicePools(yahkv.geometry(fmt, n_q, n_kv, hd, pt, g.n_pages), fill=0x5A)
    t = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")
    pos = np.asarray(starts)[:, None] + np.arange(new) + far
    r = make(yahkv, dim, layout, "yarn", first_dim=first, normalise=True)
    k_out = torch.full((n, new, n_kv, hd), float("nan"), device="cuda")
    q_out = yahkv.rotary_append(dev, t(table), t(starts), r, x[:, :, n_q:n_q + n_kv], x[:, :, n_q + n_kv:], x[:, :, :n_q],
                                positions=t(pos) if far else None, k_out=k_out, n_valid=None if n_valid is None else t(n_valid))
    torch.cuda.synchronize()
    return g, table, x, dev, pos, k_out, q_out


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("fmt,n_q,n_kv,hd,pt,starts,new,dim,first,far", [
    (8, 24, 4, 256, 64, [0, 37, 63], 1, 256, 0, 900000), (4, 8, 2, 128, 16, [15, 16, 0], 1, 64, 64, 12345),
    (8, 8, 8, 128, 32, [0, 5, 100], 7, 128, 0, 0), (8, 8, 1, 256, 16, [3, 0, 40], 21, 64, 4, 70000),
    (4, 32, 8, 128, 64, [0, 1, 64], 130, 32, 0, 500), (8, 24, 4, 256, 64, [10, 0, 64], 530, 64, 0, 100000)])
def test_append(yahkv, torch_gpu, fmt, n_q, n_kv, hd, pt, starts, new, dim, first, far, layout):
    """The rows against the definition; the pools bit for bit the oracle's quantization of the kernel's own rotated rows; rows
    of a padded chunk and everything else in the pools as they were."""
    torch = torch_gpu
    nv = [new, max(new // 2, 1), new] if new > 1 else None
    src = torch.bfloat16 if fmt == 8 else torch.float16
    g, table, x, dev, pos, k_out, q_out = append_case(yahkv, torch, fmt, n_q, n_kv, hd, pt, starts, new, layout, dim, first, src,
                                                       new + hd, nv, far)
    x64 = x.double().cpu().numpy()
    want_q = want_rows(x64[:, :, :n_q], pos, dim, layout, "yarn", first, normalise=True)
    want_k = want_rows(x64[:, :, n_q:n_q + n_kv], pos, dim, layout, "yarn", first, normalise=True)
    valid = nv or [new] * 3
    for s in range(3):
        close(torch, q_out[s, :valid[s]], want_q[s, :valid[s]], torch.float32)
        close(torch, k_out[s, :valid[s]], want_k[s, :valid[s]], torch.float32)
        assert torch.isnan(k_out[s, valid[s]:]).all()
    host = oracle.HostPools(g, fill=0x5A)
    oracle.append(host, table, starts, valid, np.nan_to_num(k_out.cpu().numpy()), np.ascontiguousarray(x64[:, :, n_q + n_kv:], np.float32))
    got = dev.numpy()
    for name, want in host.arrays().items():
        assert np.array_equal(got[name], want), name


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("fmt,n_kv,hd,pt,dim,first,src", [(8, 4, 256, 64, 256, 0, "bfloat16"), (8, 8, 128, 16, 64, 64, "float16"),
                                                          (4, 1, 256, 32, 64, 12, "float32"), (4, 2, 128, 64, 128, 0, "bfloat16")])
def test_chunk_without_rotated_rows_leaves_the_same_pools(yahkv, torch_gpu, fmt, n_kv, hd, pt, dim, first, src, layout):
    """K turned page by page (no k_out asked for) and token by token: the same operations on the same values, the same bytes,
    also where a chunk is padded, starts inside a page or runs into the end of the table (the last token owns that slot)."""
    torch = torch_gpu
    rng = np.random.default_rng(hd + dim)
    starts, new, valid = [0, 5, pt - 1, 2 * pt + 3], 77, [77, 9, 60, 77]
    pages = [(s + new + pt - 1) // pt for s in starts]
    g = yahkv.geometry(fmt, n_kv, n_kv, hd, pt, sum(pages) + 4)
    t = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")
    table = t(make_tables(rng, pages, g.n_pages))
    cut = t(np.array([0, 0, 0, table.shape[1] * pt - 50]))
    x = torch.from_numpy(rng.standard_normal((4, new, 2 * n_kv + 1, hd)).astype(np.float32)).cuda().to(getattr(torch, src))
    r = make(yahkv, dim, layout, "bands", first_dim=first, normalise=dim != 64, k_weight=torch.rand(hd, device="cuda") + 0.5)
    for start in (t(starts), cut):
        a, b = yahkv.DevicePools(g, fill=0x33), yahkv.DevicePools(g, fill=0x33)
        pos = t(rng.integers(0, 100000, (4, new)))
        k, v = x[:, :, :n_kv], x[:, :, n_kv:2 * n_kv]
        yahkv.rotary_append(a, table, start, r, k, v, positions=pos, n_valid=t(valid), k_out=torch.empty(k.shape, device="cuda"))
        yahkv.rotary_append(b, table, start, r, k, v, positions=pos, n_valid=t(valid))
        for name in ("kq", "ks", "vq", "vs"):
            assert torch.equal(getattr(a, name), getattr(b, name)), name


@pytest.mark.parametrize("n,new,pt", [(1, 130, 16), (2, 257, 32), (1, 300, 16)])
def test_long_chunk_of_few_tokens_with_rotated_rows(yahkv, torch_gpu, n, new, pt):
    """Chunks long enough to be dealt to the XCDs by pages and short enough for several workgroups a token."""
    torch = torch_gpu
    gen = torch.Generator(device="cuda").manual_seed(new)
    pages = new // pt + 2
    g = yahkv.geometry(8, 8, 2, 128, pt, n * pages)
    table = torch.randperm(n * pages, generator=gen, device="cuda").to(torch.int32).view(n, pages)
    start = torch.tensor([5, 0][:n], dtype=torch.int32, device="cuda")
    pos = torch.randint(0, 100000, (n, new), generator=gen, device="cuda", dtype=torch.int32)
    x = torch.randn(n, new, 12, 128, generator=gen, device="cuda").half()
    q, k, v = x[:, :, :8], x[:, :, 8:10], x[:, :, 10:]
    r = make(yahkv, 64, "interleaved", "ntk", first_dim=32, normalise=True)
    a, b = yahkv.DevicePools(g, fill=9), yahkv.DevicePools(g, fill=9)
    k_out = torch.full(k.shape, float("nan"), device="cuda")
    qa = yahkv.rotary_append(a, table, start, r, k, v, q, positions=pos, k_out=k_out)
    qb = yahkv.rotary_append(b, table, start, r, k, v, q, positions=pos)
    assert torch.equal(qa, qb)
    for name in ("kq", "ks", "vq", "vs"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name
    want = want_rows(k.double().cpu().numpy(), pos.cpu().numpy(), 64, "interleaved", "ntk", 32, normalise=True)
    close(torch, k_out, want, torch.float32)


def test_append_without_queries_or_norm_equals_rotate_then_append(yahkv, torch_gpu):
    torch = torch_gpu
    rng = np.random.default_rng(4)
    g = yahkv.geometry(8, 8, 2, 128, 16, 8)
    table = torch.from_numpy(rng.permutation(8).astype(np.int32).reshape(2, 4)).cuda()
    start = torch.tensor([3, 0], dtype=torch.int32, device="cuda")
    pos = torch.tensor([[70000, 5], [9, 2 ** 30]], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(2, 2, 2, 128, device="cuda") for _ in range(2))
    r = make(yahkv, 96, "interleaved", "bands", first_dim=32)
    a, b = yahkv.DevicePools(g), yahkv.DevicePools(g)
    k_out = torch.empty_like(k)
    assert yahkv.rotary_append(a, table, start, r, k, v, positions=pos, k_out=k_out) is None
    _, rows = yahkv.rotary_rows(r, pos, k=k)
    # the two kernels may contract a product and a sum differently: one rounding apart
    assert (rows - k_out).abs().max() <= 4 * 2.0 ** -24 * k.abs().max()
    yahkv.append(b, table, start, k_out, v)
    for name in ("kq", "ks", "vq", "vs"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name


def test_many_short_sequences_equal_few(yahkv, torch_gpu):
    """1200 tokens in one call and in two: the same bytes, query rows and rotated K rows."""
    torch = torch_gpu
    n, new, pt = 300, 4, 16
    gen = torch.Generator(device="cuda").manual_seed(5)
    g = yahkv.geometry(8, 24, 4, 256, pt, n)
    whole, parts = yahkv.DevicePools(g, fill=1), yahkv.DevicePools(g, fill=1)
    qkv = torch.randn(n, new, 32, 256, generator=gen, device="cuda").half()
    q, k, v = qkv[:, :, :24], qkv[:, :, 24:28], qkv[:, :, 28:]
    table = torch.randperm(n, generator=gen, device="cuda").to(torch.int32).view(n, 1)
    start = torch.randint(0, 13, (n,), generator=gen, device="cuda", dtype=torch.int32)
    pos = torch.randint(0, 100000, (n, new), generator=gen, device="cuda", dtype=torch.int32)
    r = make(yahkv, 64, "half", "linear", normalise=True)
    k_out = [torch.zeros(n, new, 4, 256, device="cuda") for _ in range(2)]
    want = yahkv.rotary_append(whole, table, start, r, k, v, q, positions=pos, k_out=k_out[0])
    half = [yahkv.rotary_append(parts, table[s], start[s], r, k[s], v[s], q[s], positions=pos[s], k_out=k_out[1][s])
            for s in (slice(0, 150), slice(150, 300))]
    assert torch.equal(want, torch.cat(half)) and torch.equal(k_out[0], k_out[1])
    for name in ("kq", "ks", "vq", "vs"):
        assert torch.equal(getattr(whole, name), getattr(parts, name)), name


def test_replays_from_a_graph_on_another_stream(yahkv, torch_gpu):
    torch = torch_gpu
    g = yahkv.geometry(8, 24, 4, 256, 64, 4)
    table = torch.arange(4, dtype=torch.int32, device="cuda").reshape(4, 1)
    start = torch.tensor([0, 5, 63, 7], dtype=torch.int32, device="cuda")
    pos = torch.tensor([[1], [2], [3], [99999]], dtype=torch.int32, device="cuda")
    x = torch.randn(4, 1, 32, 256, device="cuda").to(torch.bfloat16)
    r = make(yahkv, 64, "half", "yarn", normalise=True)
    dev = yahkv.DevicePools(g)
    q_out = torch.empty(4, 1, 24, 256, device="cuda", dtype=torch.bfloat16)
    step = lambda: yahkv.rotary_append(dev, table, start, r, x[:, :, 24:28], x[:, :, 28:], x[:, :, :24], positions=pos, q_out=q_out)
    step()
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            step()
    for i in range(3):
        x.copy_(torch.randn(4, 1, 32, 256, device="cuda"))
        pos.add_(1)
        step()
        want = [t.clone() for t in (q_out, dev.kq, dev.ks, dev.vq, dev.vs)]
        for t in (q_out, dev.kq, dev.ks, dev.vq, dev.vs):
            t.zero_() if t is not q_out else t.fill_(float("nan"))
        graph.replay()
        first = [t.clone() for t in (q_out, dev.kq, dev.ks, dev.vq, dev.vs)]
        assert torch.equal(first[0], want[0]), i
        dev.kq.zero_(), dev.ks.zero_(), dev.vq.zero_(), dev.vs.zero_()
        step()
        for name, t in zip(("kq", "ks", "vq", "vs"), first[1:]):
            assert torch.equal(getattr(dev, name), t), name
