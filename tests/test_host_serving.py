"""What the serving operators (rotary positions, shared prefixes, eviction) do on the host alone: the rotary frequency table
against exact fractions, workspace sizes, and every refusal, before anything could be launched."""
import ctypes as C
import math
from fractions import Fraction

import numpy as np
import pytest

P = 1 << 20          # an aligned address that is never followed: every call below is refused before a launch
ARG, SHAPE, WORKSPACE = -1, -2, -4


def table(yahkv, dim, scaling=0, theta=1e4, factor=8.0, length=4096.0, low=1.0, high=32.0):
    spec = yahkv.RotarySpec(dim, scaling, theta, factor, length, low, high)
    turns, mag = np.zeros(max(dim // 2, 1), np.uint64), C.c_float(-1)
    rc = yahkv.lib.yahkv_rotary_table(C.byref(spec), turns.ctypes.data, C.byref(mag))
    return rc, turns, mag.value


def frequencies(dim, scaling, theta, factor, length, low, high):
    """The scaling rules of include/yahkv.h, one pair at a time."""
    if scaling == 2:
        theta *= factor ** (dim / (dim - 2))
    got = []
    edge = lambda n: dim * math.log(length / (n * 2 * math.pi)) / (2 * math.log(theta))
    for p in range(dim // 2):
        f = theta ** (-2 * p / dim)
        if scaling == 1:
            f /= factor
        elif scaling == 3:
            a, b = max(math.floor(edge(high)), 0), min(math.ceil(edge(low)), dim - 1)
            x = min(1, max(0, (p - a) / max(b - a, 0.001)))
            f = f / factor * x + f * (1 - x)
        elif scaling == 4:
            n = length * f / (2 * math.pi)
            x = min(1, max(0, (n - low) / (high - low)))
            f = f / factor * (1 - x) + f * x
        got.append(f)
    return np.array(got)


@pytest.mark.parametrize("scaling", range(5))
@pytest.mark.parametrize("dim,theta", [(8, 1e4), (64, 1e6), (128, 5e5), (256, 1e7), (512, 1.5)])
def test_rotary_table(yahkv, dim, theta, scaling):
    low, high = (1.0, 4.0) if scaling == 4 else (1.0, 32.0)
    rc, turns, mag = table(yahkv, dim, scaling, theta, 8.0, 32768.0, low, high)
    assert rc == 0
    want = frequencies(dim, scaling, theta, 8.0, 32768.0, low, high) / (2 * math.pi)
    # pow, log and four roundings of doubles, each within a few 2^-53, and the entry's own rounding to a whole number of
    # 2^-64 turns, which is half of one of those (a slow pair has few of them: 4e10 at theta 1e7)
    assert np.all(np.abs(turns.astype(np.float64) * 2.0 ** -64 - want) < want * 64 * 2.0 ** -53 + 2.0 ** -65)
    assert mag == np.float32(0.1 * math.log(8.0) + 1) if scaling == 3 else mag == 1.0


def test_rotary_table_keeps_far_positions_exact(yahkv):
    """pos * turns modulo 2^64 is the angle's fraction of a turn: against rational arithmetic on the table's own entries."""
    _, turns, _ = table(yahkv, 64, 0, 1e7)
    for pos in (0, 1, -1, 10 ** 6, 2 ** 31 - 1, -2 ** 31):
        for f in turns[[0, 1, 17, 31]]:
            exact = Fraction(pos) * Fraction(int(f), 2 ** 64) % 1
            assert Fraction(pos * int(f) % 2 ** 64, 2 ** 64) == exact


def exact_turns(dim, scaling, theta, factor, length, low, high):
    """The frequencies of include/yahkv.h in turns, to 60 decimal digits."""
    from decimal import Decimal as D, ROUND_CEILING, ROUND_FLOOR, localcontext
    with localcontext() as c:
        c.prec = 60
        pi2 = D("6.28318530717958647692528676655900576839433879875021164194988918461563281257")
        theta, factor, length, low, high = D(theta), D(factor), D(length), D(low), D(high)
        if scaling == 2:
            theta *= (factor.ln() * dim / (dim - 2)).exp()
        edge = lambda n: dim * (length / (n * pi2)).ln() / (2 * theta.ln())
        a = max(edge(high).to_integral_value(ROUND_FLOOR), D(0))
        b = min(edge(low).to_integral_value(ROUND_CEILING), D(dim - 1))
        got = []
        for p in range(dim // 2):
            f = (theta.ln() * -2 * p / dim).exp()
            if scaling == 1:
                f /= factor
            elif scaling == 3:
                x = min(D(1), max(D(0), (p - a) / max(b - a, D(0.001))))
                f = f / factor * x + f * (1 - x)
            elif scaling == 4:
                x = min(D(1), max(D(0), (length * f / pi2 - low) / (high - low)))
                f = f / factor * (1 - x) + f * x
            got.append(f / pi2)
        return got


@pytest.mark.parametrize("scaling", range(5))
@pytest.mark.parametrize("dim,theta", [(8, 1e4), (64, 1e4), (64, 1e7), (72, 1e6), (128, 5e5), (256, 1e7), (512, 1.5)])
def test_rotary_table_to_its_last_bits(yahkv, dim, theta, scaling):
    """Every entry within two of its units, 2^-63 turns: half of one is its own rounding, and the operations before it, in 64 bits
    of significand, err by a few 2^-64 of a frequency that is 2^61.4 units at most (powers one step of 2^-63, its exponent,
    quotients and products half of one each, and the ramp of the banded rules up to twice as many: 8 x 2^-64 x 2^61.4 = 1.4)."""
    from decimal import Decimal as D
    low, high = (1.0, 4.0) if scaling == 4 else (1.0, 32.0)
    rc, turns, _ = table(yahkv, dim, scaling, theta, 8.0, 32768.0, low, high)
    assert rc == 0
    off = [abs(D(int(t)) - w * 2 ** 64) for t, w in zip(turns, exact_turns(dim, scaling, theta, 8.0, 32768.0, low, high))]
    assert max(off) <= 2, float(max(off))


@pytest.mark.parametrize("change", [dict(dim=4), dict(dim=0), dict(dim=-8), dict(dim=12), dict(theta=1.0), dict(theta=float("nan")),
                                    dict(theta=float("inf")), dict(scaling=5), dict(scaling=-1), dict(scaling=1, factor=0.5),
                                    dict(scaling=1, factor=float("nan")), dict(scaling=3, length=0.0), dict(scaling=4, low=0.0),
                                    dict(scaling=4, low=4.0, high=4.0), dict(scaling=3, high=float("inf")),
                                    dict(scaling=2, factor=float("inf"))])
def test_rotary_table_refusals(yahkv, change):
    assert table(yahkv, **dict(dict(dim=64), **change))[0] == ARG


def test_rotary_table_null(yahkv):
    assert yahkv.lib.yahkv_rotary_table(None, None, None) == ARG


def rotary(yahkv, **kw):
    f = dict(turns=P, rotary_dim=64, first_dim=0, layout=0, magnitude=1.0, normalise=0, eps=1e-6, q_weight=None, k_weight=None)
    f.update(kw)
    return yahkv.RotaryStruct(*f.values())


def rows(yahkv, heads, d=128, **kw):
    f = dict(data=P, dtype=2, n_heads=heads, seq_stride=heads * d, token_stride=heads * d, head_stride=d)
    f.update(kw)
    return yahkv.Rows(*f.values())


def apply(yahkv, r=None, d=128, pos=P, n=1, new=1, **kw):
    q = {k: kw[k] for k in kw}
    a = dict(qs=rows(yahkv, 8), qd=rows(yahkv, 8), ks=rows(yahkv, 2), kd=rows(yahkv, 2))
    a.update(q)
    ref = lambda s: None if s is None else C.byref(s)
    return yahkv.lib.yahkv_rotary_apply(ref(r or rotary(yahkv)), d, pos, n, new, ref(a["qs"]), ref(a["qd"]), ref(a["ks"]), ref(a["kd"]), None)


def test_rotary_apply_refusals(yahkv):
    for kw in (dict(turns=None), dict(turns=P + 4), dict(rotary_dim=4), dict(rotary_dim=12), dict(rotary_dim=136), dict(rotary_dim=0),
               dict(first_dim=-4), dict(first_dim=2), dict(first_dim=68), dict(layout=2), dict(normalise=1, eps=-1.0),
               dict(normalise=1, eps=float("nan")), dict(q_weight=P + 4), dict(k_weight=P + 8)):
        assert apply(yahkv, rotary(yahkv, **kw)) == ARG, kw
    for kw in (dict(data=None), dict(data=P + 8), dict(dtype=3), dict(n_heads=0), dict(n_heads=7), dict(seq_stride=4), dict(token_stride=2),
               dict(head_stride=12), dict(dtype=0, head_stride=2)):
        assert apply(yahkv, qs=rows(yahkv, 8, **kw)) == ARG, kw
        assert apply(yahkv, kd=rows(yahkv, 2, **kw)) == ARG, kw
    assert apply(yahkv, qs=rows(yahkv, 8, dtype=1)) == ARG               # q and k of two types
    assert apply(yahkv, qd=None) == ARG and apply(yahkv, ks=None) == ARG
    assert apply(yahkv, qs=None, qd=None, ks=None, kd=None) == ARG
    assert apply(yahkv, pos=None) == ARG and apply(yahkv, n=0) == ARG and apply(yahkv, new=-1) == ARG
    for d in (0, 4, 130, 520):
        assert apply(yahkv, d=d) == SHAPE
    assert apply(yahkv, n=1 << 20, new=1 << 20) == SHAPE


def test_destination_rows_at_one_address_are_refused(yahkv):
    for kw in (dict(seq_stride=0), dict(token_stride=0), dict(head_stride=0)):
        assert apply(yahkv, n=2, new=2, qd=rows(yahkv, 8, **kw)) == ARG, kw
        assert apply(yahkv, n=2, new=2, kd=rows(yahkv, 2, **kw)) == ARG, kw
    g = yahkv.geometry(8, 8, 2, 128, 16, 4)
    k, v, q, out = rows(yahkv, 2), rows(yahkv, 2), rows(yahkv, 8), rows(yahkv, 8, token_stride=0)
    assert yahkv.lib.yahkv_rotary_append(C.byref(g), C.byref(pools(yahkv, g)), P, 4, P, None, 1, 9, C.byref(rotary(yahkv)), None,
                                         C.byref(k), C.byref(v), C.byref(q), C.byref(out), None, None) == ARG


def pools(yahkv, g, **kw):
    b = yahkv.pool_bytes(g)
    f = dict(kq=P, ks=P, vq=P, vs=P, kq_bytes=b["kq"], ks_bytes=b["ks"], vq_bytes=b["vq"], vs_bytes=b["vs"])
    f.update(kw)
    return yahkv.Pools(*f.values())


def test_rotary_append_refusals(yahkv):
    g = yahkv.geometry(8, 8, 2, 128, 16, 4)

    def call(g=g, p=None, tab=P, stride=4, start=P, n=1, new=1, r=None, k="k", v="v", qs=None, qd=None, k_out=None):
        k = rows(yahkv, 2) if k == "k" else k
        v = rows(yahkv, 2) if v == "v" else v
        ref = lambda s: None if s is None else C.byref(s)
        return yahkv.lib.yahkv_rotary_append(C.byref(g), C.byref(p or pools(yahkv, g)), tab, stride, start, None, n, new,
                                             ref(r or rotary(yahkv)), None, ref(k), ref(v), ref(qs), ref(qd), k_out, None)
    assert call(k=None) == ARG and call(v=None) == ARG and call(tab=None) == ARG and call(start=None) == ARG
    assert call(n=0) == ARG and call(new=0) == ARG and call(stride=0) == ARG
    assert call(k=rows(yahkv, 1)) == ARG and call(v=rows(yahkv, 2, dtype=1)) == ARG and call(k=rows(yahkv, 2, data=P + 8)) == ARG
    assert call(v=rows(yahkv, 2, head_stride=4)) == ARG
    assert call(qs=rows(yahkv, 8)) == ARG and call(qd=rows(yahkv, 8)) == ARG
    assert call(qs=rows(yahkv, 4), qd=rows(yahkv, 4)) == ARG and call(qs=rows(yahkv, 8, dtype=0), qd=rows(yahkv, 8)) == ARG
    assert call(r=rotary(yahkv, rotary_dim=256)) == ARG and call(k_out=P + 4) == ARG
    assert call(p=pools(yahkv, g, vq_bytes=16)) == ARG and call(p=pools(yahkv, g, ks=None)) == ARG
    assert call(g=yahkv.f16_geometry(8, 2, 128, 16, 4), p=pools(yahkv, g)) == SHAPE
    assert call(n=1 << 16, new=1 << 16) == SHAPE


def test_shared_refusals(yahkv):
    g = yahkv.geometry(8, 8, 2, 128, 16, 64)
    size = yahkv.decode_shared_workspace_bytes(g, 4, 2, 256, 64)
    assert size > 0
    for bad in ((0, 1, 256, 64), (4, 0, 256, 64), (4, 5, 256, 64), (4, 2, -1, 64), (4, 2, 256, 0), (9000, 1, 256, 64)):
        assert yahkv.decode_shared_workspace_bytes(g, *bad) == 0
    assert yahkv.decode_shared_workspace_bytes(g, 4, 2, 0, 64) > 0        # no prefix at all is a plain decode

    def call(g=g, p=None, tab=P, stride=64, lens=P, n=4, first=P, shared=P, groups=2, ms=256, mt=64, q=P, qt=2, scale=0.1,
             out=P, ot=0, ws=P, nbytes=size):
        return yahkv.lib.yahkv_decode_attend_shared(C.byref(g), C.byref(p or pools(yahkv, g)), tab, stride, lens, n, first, shared,
                                                    groups, ms, mt, q, qt, scale, None, out, ot, ws, nbytes, None)
    for kw in (dict(tab=None), dict(lens=None), dict(first=None), dict(shared=None), dict(q=None), dict(out=None), dict(ws=None),
               dict(stride=0), dict(n=0), dict(groups=0), dict(groups=5), dict(ms=-1), dict(mt=0), dict(q=P + 8), dict(out=P + 4),
               dict(ws=P + 8), dict(qt=3), dict(ot=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
               dict(p=pools(yahkv, g, kq_bytes=1))):
        assert call(**kw) == ARG, kw
    assert call(nbytes=size - 1) == WORKSPACE and call(n=9000) == SHAPE
    assert call(stride=1 << 28) == SHAPE                                  # positions beyond 31 bits
    assert call(g=yahkv.f16_geometry(8, 2, 128, 16, 64), p=pools(yahkv, g)) == SHAPE


def test_weights_refusals(yahkv):
    g = yahkv.geometry(4, 8, 2, 128, 16, 64)
    size = yahkv.decode_weights_workspace_bytes(g, 3, 500)
    assert size > 0 and yahkv.decode_weights_workspace_bytes(g, 0, 500) == 0 and yahkv.decode_weights_workspace_bytes(g, 3, 0) == 0

    def call(p=None, tab=P, stride=64, lens=P, n=3, longest=500, q=P, qt=1, out=P, ot=1, win=P, wout=P, ws_stride=500, ws=P, nbytes=size):
        return yahkv.lib.yahkv_decode_attend_weights(C.byref(g), C.byref(p or pools(yahkv, g)), tab, stride, lens, n, longest, q, qt, 0.1,
                                                     None, out, ot, win, wout, ws_stride, 1.0, ws, nbytes, None)
    for kw in (dict(tab=None), dict(lens=None), dict(n=0), dict(longest=0), dict(q=None), dict(q=P + 2), dict(qt=7), dict(out=None),
               dict(out=P + 8), dict(ot=3), dict(wout=None), dict(ws_stride=499), dict(ws=None), dict(ws=P + 4), dict(stride=0),
               dict(p=pools(yahkv, g, vs=P + 8))):
        assert call(**kw) == ARG, kw
    assert call(nbytes=size - 1) == WORKSPACE and call(n=9000) == SHAPE


def test_evict_refusals(yahkv):
    g = yahkv.geometry(8, 8, 2, 128, 16, 64)

    def select(lens=P, n=3, longest=500, w=P, ws=500, budget=100, sink=4, recent=32, kept=P, n_kept=P):
        return yahkv.lib.yahkv_evict_select(C.byref(g), lens, n, longest, w, ws, budget, sink, recent, kept, n_kept, None)
    for kw in (dict(lens=None), dict(w=None), dict(kept=None), dict(n_kept=None), dict(n=0), dict(longest=0), dict(ws=499), dict(budget=0),
               dict(sink=-1), dict(recent=-1), dict(sink=50, recent=51), dict(sink=2 ** 31 - 1, recent=2 ** 31 - 1)):
        assert select(**kw) == ARG, kw
    assert select(n=70000) == SHAPE

    def compact(p=None, tab=P, stride=32, kept=P, n_kept=P, n=3, budget=100, dst=P + 16, ds=7, wi=P, wis=500, wo=P + 16, wos=100):
        return yahkv.lib.yahkv_evict_compact(C.byref(g), C.byref(p or pools(yahkv, g)), tab, stride, kept, n_kept, n, budget, dst, ds, wi, wis,
                                             wo, wos, None)
    for kw in (dict(tab=None), dict(kept=None), dict(n_kept=None), dict(dst=None), dict(dst=P), dict(n=0), dict(budget=0), dict(stride=0),
               dict(ds=6), dict(wi=None), dict(wo=None), dict(wis=0), dict(wos=99), dict(wo=P), dict(p=pools(yahkv, g, kq=P + 8))):
        assert compact(**kw) == ARG, kw
    assert compact(n=70000) == SHAPE and compact(stride=1 << 28) == SHAPE


def test_binding_refuses_tensors_of_another_shape(yahkv):
    """Shapes and types that the C entry points would take on trust."""
    import torch
    g = yahkv.geometry(8, 8, 2, 128, 16, 4)
    dev = yahkv.DevicePools(g, device="cpu")
    i = lambda *s: torch.zeros(s, dtype=torch.int32)
    q = torch.zeros(3, 8, 128)
    tab = i(3, 4)
    for bad in (dict(seq_len=i(2)), dict(group_first=i(1)), dict(shared_len=i(1, 1)), dict(table=i(2, 4)), dict(q=q[:, :4]),
                dict(seq_len=i(3).long()), dict(out=torch.zeros(3, 8, 64)), dict(gate=torch.zeros(3, 8, 1)), dict(table=i(4, 3).t())):
        a = dict(table=tab, seq_len=i(3), group_first=i(2), shared_len=i(1), max_shared_len=64, max_tail_len=64, q=q, scale=0.1)
        a.update(bad)
        with pytest.raises(yahkv.YahkvError):
            yahkv.decode_attend_shared(dev, **a)
    for bad in (dict(weights_out=torch.zeros(3, 2, 63)), dict(weights_out=torch.zeros(3, 8, 64)), dict(weights_in=torch.zeros(3, 2, 65)),
                dict(weights_out=torch.zeros(3, 2, 64).half())):
        a = dict(table=tab, seq_len=i(3), max_seq_len=64, q=q, scale=0.1, weights_out=torch.zeros(3, 2, 64))
        a.update(bad)
        with pytest.raises(yahkv.YahkvError):
            yahkv.decode_attend_weights(dev, **a)
    for bad in (dict(kept=i(3, 1, 8)), dict(n_kept=i(2)), dict(dst_table=i(2, 1)), dict(weights_in=torch.zeros(3, 3, 9)),
                dict(weights_in=torch.zeros(3, 2, 64), weights_out=torch.zeros(3, 2, 7))):
        a = dict(table=tab, kept=i(3, 2, 8), n_kept=i(3), dst_table=i(3, 1))
        a.update(bad)
        with pytest.raises(yahkv.YahkvError):
            yahkv.evict_compact(dev, **a)
    r = yahkv.Rotary(64, 1e4, device="cpu")
    x = torch.zeros(3, 1, 8, 128)
    for a in ((i(3), x), (i(3, 2), x), (i(3, 1).long(), x), (i(3, 1), x.transpose(2, 3)), (i(3, 1), None)):
        with pytest.raises(yahkv.YahkvError):
            yahkv.rotary_rows(r, *a)
    with pytest.raises(yahkv.YahkvError):
        yahkv.Rotary(64, 1e4, layout="neox", device="cpu")
    with pytest.raises(yahkv.YahkvError):
        yahkv.rotary_rows(yahkv.Rotary(64, 1e4, q_weight=torch.ones(64), device="cpu"), i(3, 1), x)
    with pytest.raises(yahkv.YahkvError):
        yahkv.DevicePools.of(g, dev.kq, dev.ks, dev.vq.view(2, -1).t(), dev.vs)


def test_shared_workspace_does_not_grow_with_the_bounds(yahkv):
    """Bounds far above the lengths cost a bounded number of partials: 64 rows of 16 workgroups for each of 256 compute units."""
    g = yahkv.geometry(8, 24, 4, 256, 64, 1000)
    for n, groups, shared, tail in ((1, 1, 0, 2 ** 30), (64, 1, 32768, 2 ** 30), (64, 64, 2 ** 30, 2 ** 30)):
        assert 0 < yahkv.decode_shared_workspace_bytes(g, n, groups, shared, tail) <= 64 * 16 * 256 * 258 * 4


def test_output_types_are_refused(yahkv):
    import torch
    q = torch.zeros(1, 8, 128, dtype=torch.float16)
    with pytest.raises(yahkv.YahkvError):
        yahkv._out(None, q, torch.int32, torch.float32)
    with pytest.raises(yahkv.YahkvError):
        yahkv._out(torch.zeros(1, 8, 128, dtype=torch.int32), q, None, torch.float32)
    assert yahkv._out(None, q.transpose(1, 2), torch.bfloat16, torch.float32).is_contiguous()


def test_rotary_outputs_of_another_type_than_asked_for_are_refused(yahkv):
    """(A call that passes every look at its tensors is refused for their device here.)"""
    import torch
    r = yahkv.Rotary(64, 1e4, device="cpu")
    pos, x = torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, 1, 2, 128)
    half, same = x.half(), torch.empty_like(x)
    for a in (dict(q_out=half, out_dtype=torch.float32), dict(k=x, q_out=same, k_out=half, out_dtype=torch.float32)):
        with pytest.raises(yahkv.YahkvError, match="another type"):
            yahkv.rotary_rows(r, pos, x, **a)
    for a in (dict(q_out=half), dict(q_out=half, out_dtype=torch.float16), dict(k=x, q_out=half, out_dtype=torch.float32)):
        with pytest.raises(yahkv.YahkvError, match="on a GPU"):
            yahkv.rotary_rows(r, pos, x, **a)
    g = yahkv.geometry(8, 4, 2, 128, 16, 4)
    dev, i, q = yahkv.DevicePools(g, device="cpu"), torch.zeros(3, dtype=torch.int32), torch.zeros(3, 1, 4, 128)
    for a, why in ((dict(q_out=q.half(), q_out_dtype=torch.float32), "another type"), (dict(q_out=q.half()), "on a GPU"),
                   (dict(q_out=q.half(), q_out_dtype=torch.float16), "on a GPU"), (dict(q_out_dtype=torch.float16), "on a GPU")):
        with pytest.raises(yahkv.YahkvError, match=why):
            yahkv.rotary_append(dev, torch.zeros(3, 1, dtype=torch.int32), i, r, x, x, q, **a)


@pytest.mark.parametrize("name", ["ks", "vq", "vs"])
def test_pools_on_two_devices_are_refused(yahkv, name):
    g = yahkv.geometry(8, 8, 2, 128, 16, 4)
    t = yahkv.DevicePools(g, device="cpu")
    a = dict(kq=t.kq, ks=t.ks, vq=t.vq, vs=t.vs)
    assert yahkv.DevicePools.of(g, **a).vs.data_ptr() == t.vs.data_ptr()
    with pytest.raises(yahkv.YahkvError, match="device"):
        yahkv.DevicePools.of(g, **dict(a, **{name: a[name].to("meta")}))
