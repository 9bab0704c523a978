"""What the long-context serving operators are measured on: their cases, their inputs, a plain form of each and its
definition in 64 bits.

Five operators over the block-quantized paged cache (include/yahkv.h), as one decode loop uses them:

  shared   decode attention of a batch whose sequences begin with a common prefix, held once in shared pages
  weights  decode attention that also adds each key's softmax weight to a running sum per (sequence, kv head)
  evict    the choice of the keys to keep by those sums, and the move of the kept ones to fresh pages
  rotary   rotary positions of query and key rows in either layout, on a part of the head, scaled for long contexts
  append   the same fused with the block quantization of the key and value rows into their pages

`own` false: plain torch in 32 bits (the angles of far positions in 64). `own` true: the library's entry points.
"""
import importlib
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# (query heads, kv heads, head dim): the benchmark's own layout, and grouped, plain and single-kv-head layouts
HEADS = {"24/4x256": (24, 4, 256), "32/8x128": (32, 8, 128), "8/8x128": (8, 8, 128), "8/1x256": (8, 1, 256)}


def _heads(case):
    return HEADS[case["heads"]]


# ---- cases ------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # a handful of requests that have just begun to answer one prompt: latency counts
        dict(name="shared_few", op="shared", fmt=8, heads="24/4x256", pt=64, seqs=4, groups=1, prefix=2048, tail=40,
             q="bf16", out="bf16"),
        # a service's system prompt before a batch of ordinary requests
        dict(name="shared_b32", op="shared", fmt=8, heads="24/4x256", pt=64, seqs=32, groups=1, prefix=8192, tail=700,
             q="bf16", out="bf16"),
        # three tenants' prompts of odd lengths side by side, small pages, 4-bit codes, one idle slot
        dict(name="shared_groups_q4", op="shared", fmt=4, heads="32/8x128", pt=16, seqs=45, groups=3, prefix=5003,
             tail=333, q="f16", out="f16"),
        # a long document asked about by a full batch
        dict(name="shared_b64_long", op="shared", fmt=8, heads="24/4x256", pt=64, seqs=64, groups=1, prefix=32768,
             tail=2048, q="bf16", out="f16"),
        # one long sequence whose keys are being weighed
        dict(name="weights_b1", op="weights", fmt=8, heads="24/4x256", pt=64, seqs=1, longest=32768, q="bf16", out="bf16"),
        # a ragged batch, 4-bit codes, small pages
        dict(name="weights_b24_q4", op="weights", fmt=4, heads="32/8x128", pt=16, seqs=24, longest=16001, q="f16",
             out="f16"),
        # one long sequence cut to an eighth
        dict(name="evict_b1", op="evict", fmt=8, heads="24/4x256", pt=64, seqs=1, longest=32768, budget=4096, sink=4,
             recent=512),
        # a ragged batch cut to a common budget; some sequences are shorter than it
        dict(name="evict_b32", op="evict", fmt=8, heads="24/4x256", pt=64, seqs=32, longest=16384, budget=2048, sink=4,
             recent=256),
        # one token of a full batch at far positions
        dict(name="rotary_step", op="rotary", heads="24/4x256", seqs=64, new=1, far=1000000, layout="half", rotary=256,
             scaling="yarn", normalise=True, src="bf16", out="bf16"),
        # a prefill chunk out of one fused projection, part of the head, interleaved pairs
        dict(name="rotary_chunk", op="rotary", heads="24/4x256", seqs=8, new=2048, far=16384, layout="interleaved",
             rotary=64, scaling="bands", normalise=False, src="bf16", out="bf16"),
        # one token of a full batch into its pages
        dict(name="append_step", op="append", fmt=8, heads="24/4x256", pt=16, seqs=64, new=1, far=200000, layout="half",
             rotary=64, scaling="yarn", normalise=True, src="bf16", out="bf16"),
        # an odd chunk into pages of half the size
        dict(name="append_chunk", op="append", fmt=8, heads="32/8x128", pt=32, seqs=5, new=1037, far=30000,
             layout="interleaved", rotary=128, scaling="linear", normalise=True, src="f16", out="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["shared", "weights", "evict", "rotary", "append"])
    c = dict(op=op, heads=rng.choice(sorted(HEADS)))
    d = _heads(c)[2]
    if op in ("shared", "weights", "evict"):
        c.update(fmt=rng.choice([8, 4]), pt=rng.choice([16, 32, 64]))
    if op == "shared":
        c.update(seqs=_log(rng, 1, 64))
        c.update(groups=min(c["seqs"], rng.choice([1, 1, 2, 4])), prefix=_log(rng, 30, 32768), tail=_log(rng, 1, 2048),
                 q=rng.choice(["bf16", "f16", "f32"]), out=rng.choice(["bf16", "f16"]))
    elif op == "weights":
        c.update(seqs=_log(rng, 1, 32), longest=_log(rng, 1, 32768), q=rng.choice(["bf16", "f16"]),
                 out=rng.choice(["bf16", "f16"]))
    elif op == "evict":
        c.update(seqs=_log(rng, 1, 32), longest=_log(rng, 20, 32768))
        c.update(budget=_log(rng, 8, max(9, c["longest"])), sink=rng.choice([0, 1, 4]))
        c.update(recent=rng.randint(0, c["budget"] - c["sink"]))
    else:
        new = rng.choice([1, 1, _log(rng, 2, 2048)])
        c.update(seqs=_log(rng, 1, 64 if new == 1 else 8), new=new, far=_log(rng, 10, 1000000),
                 layout=rng.choice(["half", "interleaved"]), rotary=rng.choice([d // 4, d // 2, d]),
                 scaling=rng.choice(["none", "linear", "ntk", "yarn", "bands"]), normalise=rng.random() < 0.5,
                 src=rng.choice(["bf16", "f16", "f32"]), out=rng.choice(["bf16", "f16", "f32"]))
        if op == "append":
            # (8-bit codes only: a value next to the border between two 4-bit codes may go either way, and one such step
            # is a third of a typical value)
            c.update(fmt=8, pt=rng.choice([16, 32, 64]))
    return c


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32)


def _cache(case, gen, pages):
    """Random pools of `pages` pages as a filled cache leaves them: blocks of 32 normal values, codes and f16 scales."""
    _, kv, d = _heads(case)
    pt, nb, q8 = case["pt"], d // 32, case["fmt"] == 8
    k = torch.empty(pages, kv, nb, pt, 32 if q8 else 16, dtype=torch.uint8, device=DEV)
    v = torch.empty(pages, kv, d if q8 else nb * 16, pt, dtype=torch.uint8, device=DEV)
    ks = torch.empty(pages, kv, pt, nb, dtype=torch.float16, device=DEV)
    vs = torch.empty(pages, kv, nb, pt, dtype=torch.float16, device=DEV)
    for p in range(0, pages, 512):  # in pieces: the values are four to eight times their codes
        n = min(512, pages - p)
        for codes, scales, transposed in ((k, ks, False), (v, vs, True)):
            x = _normal(gen, n, kv, nb, pt, 32)
            s = x.abs().amax(-1, keepdim=True) / (127.0 if q8 else 7.5)
            s16 = s.to(torch.float16)
            if q8:
                c = torch.round(x / s).to(torch.int8).view(torch.uint8)
            else:
                u = torch.clamp(torch.round(x / s) + 8, 0, 15).to(torch.uint8)
                c = u[..., :16] | (u[..., 16:] << 4)
            if transposed:
                codes[p:p + n] = c.permute(0, 1, 2, 4, 3).reshape(n, kv, -1, pt)
                scales[p:p + n] = s16[..., 0]
            else:
                codes[p:p + n] = c
                scales[p:p + n] = s16[..., 0].transpose(2, 3)
    return dict(kq=k, ks=ks, vq=v, vs=vs)


def _lengths(case, rng):
    """Ragged lengths spread from one token to `longest`, the same ones in another order for every seed; the first
    sequence has them all, an idle slot (if there are four) none."""
    n, top = case["seqs"], case["longest"]
    u = (np.arange(n) + 0.5) / n
    lens = np.maximum(1, np.round(np.where(np.arange(n) % 4 == 0, top ** u, top * u))).astype(np.int64)
    lens[-1] = top
    if n >= 4:
        lens[1] = 0
    lens[:-1] = rng.permutation(lens[:-1])
    return np.roll(lens, 1)


def _int(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = np.random.default_rng(seed)
    nq, kv, d = _heads(case)
    s = dict(case=case)
    if case["op"] == "shared":
        pt, n = case["pt"], case["seqs"]
        members = np.array_split(np.arange(n), case["groups"])
        first = np.cumsum([0] + [len(m) for m in members])
        shared = np.array([case["prefix"]] + [int(rng.integers(case["prefix"] // 2 + 1, case["prefix"] + 1))
                                              for _ in members[1:]])
        lens = np.zeros(n, np.int64)
        for g, m in enumerate(members):
            lens[m] = shared[g] + rng.integers(0, case["tail"] + 1, len(m))
            lens[m[0]] = shared[g] + case["tail"]
        if n >= 40:
            lens[n // 2] = 0  # an idle slot
        whole = shared // pt  # a prefix's full pages are shared, its last, partly filled page is everybody's own
        stride = int(-(-lens.max() // pt))
        need = [-(-int(l) // pt) for l in lens]
        own_pages = sum(max(0, need[i] - int(whole[g])) for g, m in enumerate(members) for i in m)
        total = int(whole.sum()) + own_pages
        perm = rng.permutation(total)
        table, at = np.zeros((n, stride), np.int64), 0
        for g, m in enumerate(members):
            common = perm[at:at + whole[g]]
            at += whole[g]
            for i in m:
                table[i, :whole[g]] = common
                mine = max(0, need[i] - int(whole[g]))
                table[i, whole[g]:whole[g] + mine] = perm[at:at + mine]
                at += mine
        s.update(_cache(case, gen, total), pages=total, table=_int(table), seq_len=_int(lens), max_len=int(lens.max()),
                 group_first=_int(first), shared_len=_int(shared), max_shared=int(shared.max()),
                 max_tail=int(max((lens[m] - shared[g] // 64 * 64).max() for g, m in enumerate(members))))
        s["max_tail"] = max(1, s["max_tail"])
        s["q"] = (_normal(gen, n, nq, d) * 2.0).to(DTYPES[case["q"]])  # scores with a standard deviation of two
        s["scale"] = 1.0 / math.sqrt(d)
    elif case["op"] in ("weights", "evict"):
        pt, n = case["pt"], case["seqs"]
        lens = _lengths(case, rng)
        need = -(-lens // pt)
        stride = int(max(1, need.max()))
        budget_pages = -(-case["budget"] // pt) if case["op"] == "evict" else 0
        total = int(need.sum()) + n * budget_pages
        perm = rng.permutation(total)
        table, at = np.zeros((n, stride), np.int64), 0
        for i in range(n):
            table[i, :need[i]] = perm[at:at + need[i]]
            at += int(need[i])
        s.update(_cache(case, gen, total), pages=total, table=_int(table), seq_len=_int(lens), max_len=int(lens.max()))
        # sums over some steps: a few keys carry most of the weight, most carry little
        w = torch.exp(_normal(gen, n, kv, s["max_len"]) * 2.0) * (10.0 / s["max_len"])
        s["weights"] = w
        if case["op"] == "weights":
            s["q"] = (_normal(gen, n, nq, d) * 2.0).to(DTYPES[case["q"]])
            s["scale"] = 1.0 / math.sqrt(d)
            s["weights_out"] = torch.zeros_like(w)
        else:
            s["dst_table"] = _int(perm[at:].reshape(n, budget_pages))
            s["weights_out"] = torch.zeros(n, kv, case["budget"], dtype=torch.float32, device=DEV)
    else:
        n, new = case["seqs"], case["new"]
        heads = nq + 2 * kv
        # one fused projection's output, as a layer hands it over: query, key and value rows side by side
        x = _normal(gen, n, new, heads * d).to(DTYPES[case["src"]])
        s["qkv"] = x.view(n, new, heads, d)
        start = rng.integers(0, case["far"] + 1, n)
        s["positions"] = _int(start[:, None] + np.arange(new)[None])
        s["qw"] = 1.0 + 0.1 * _normal(gen, d)
        s["kw"] = 1.0 + 0.1 * _normal(gen, d)
        s["spec"] = dict(rotary_dim=case["rotary"], theta=1e7 if case["scaling"] != "bands" else 5e5,
                         scaling=case["scaling"], factor=8.0 if case["scaling"] != "none" else 1.0, original_len=32768.0,
                         **(dict(low=1.0, high=4.0) if case["scaling"] == "bands" else dict(low=1.0, high=32.0)))
        if case["op"] == "append":
            pt = case["pt"]
            slot0 = rng.integers(0, 2 * pt, n)  # where in its cache each sequence stands (its keys may have been thinned out)
            need = -(-(slot0 + new) // pt)
            most = -(-(2 * pt - 1 + new) // pt)
            total = n * most
            perm, at = rng.permutation(total), 0
            table = np.zeros((n, most), np.int64)
            for i in range(n):
                table[i, :need[i]] = perm[at:at + need[i]]
                at += int(need[i])
            s.update(_cache(case, gen, total), pages=total, table=_int(table), start=_int(slot0))
    return s


# ---- the framework's calls ----------------------------------------------------------------------------------------------

def _held(s, name, make):
    """What a program makes once and keeps beside its tensors (the pools' handle, the frequency table, a workspace)."""
    if name not in s:
        s[name] = make()
    return s[name]


def _pools(s, lib):
    c = s["case"]
    return _held(s, "pools", lambda: lib.DevicePools.of(
        lib.geometry(c["fmt"], *_heads(c), c["pt"], s["pages"]), s["kq"], s["ks"], s["vq"], s["vs"]))


def _rotary(s, lib):
    c, p = s["case"], s["spec"]
    return _held(s, "rotary", lambda: lib.Rotary(
        c["rotary"], p["theta"], layout=c["layout"], scaling=p["scaling"], factor=p["factor"],
        original_len=p["original_len"], low=p["low"], high=p["high"], normalise=c["normalise"], eps=1e-6,
        q_weight=s["qw"] if c["normalise"] else None, k_weight=s["kw"] if c["normalise"] else None, device=DEV))


def _run_own(s):
    lib = importlib.import_module("yet-another-halo-engine_amd")
    c = s["case"]
    op = c["op"]
    nq, kv, _ = _heads(c)
    if op == "shared":
        pools = _pools(s, lib)
        ws = _held(s, "ws", lambda: torch.empty(lib.decode_shared_workspace_bytes(
            pools.geom, c["seqs"], c["groups"], s["max_shared"], s["max_tail"]), dtype=torch.uint8, device=DEV))
        return lib.decode_attend_shared(pools, s["table"], s["seq_len"], s["group_first"], s["shared_len"],
                                        s["max_shared"], s["max_tail"], s["q"], s["scale"], out_dtype=DTYPES[c["out"]],
                                        workspace=ws)
    if op == "weights":
        pools = _pools(s, lib)
        ws = _held(s, "ws", lambda: torch.empty(lib.decode_weights_workspace_bytes(
            pools.geom, c["seqs"], s["max_len"]), dtype=torch.uint8, device=DEV))
        out = lib.decode_attend_weights(pools, s["table"], s["seq_len"], s["max_len"], s["q"], s["scale"],
                                        s["weights_out"], weights_in=s["weights"], out_dtype=DTYPES[c["out"]], workspace=ws)
        return out, s["weights_out"]
    if op == "evict":
        pools = _pools(s, lib)
        kept, n_kept = lib.evict_select(pools.geom, s["seq_len"], s["max_len"], s["weights"], c["budget"], c["sink"],
                                        c["recent"])
        lib.evict_compact(pools, s["table"], kept, n_kept, s["dst_table"], s["weights"], s["weights_out"])
        return kept, n_kept, s["weights_out"], s["kq"], s["ks"], s["vq"], s["vs"]
    x = s["qkv"]
    q, k, v = x[:, :, :nq], x[:, :, nq:nq + kv], x[:, :, nq + kv:]
    rot = _rotary(s, lib)
    if op == "rotary":
        return lib.rotary_rows(rot, s["positions"], q, k, out_dtype=DTYPES[c["out"]])
    pools = _pools(s, lib)
    q_out = lib.rotary_append(pools, s["table"], s["start"], rot, k, v, q, positions=s["positions"],
                              q_out_dtype=DTYPES[c["out"]])
    return (q_out,) + _values16(s)


# ---- the plain forms ------------------------------------------------------------------------------------------------------

def _k_values(c, kq, ks):
    """K codes [.., H, NB, PT, 32 | 16] and scales [.., H, PT, NB] as f32 [.., H, PT, D]."""
    if c["fmt"] == 8:
        x = kq.view(torch.int8).float()
    else:
        x = torch.cat([kq & 15, kq >> 4], -1).float() - 8.0
    x = x * ks.float().transpose(-1, -2).unsqueeze(-1)
    x = x.transpose(-3, -2)
    return x.reshape(*x.shape[:-2], -1)


def _v_values(c, vq, vs):
    """V codes [.., H, D | NB * 16, PT] and scales [.., H, NB, PT] as f32 [.., H, PT, D]."""
    nb, pt = vs.shape[-2], vs.shape[-1]
    x = vq.reshape(*vq.shape[:-2], nb, -1, pt)
    if c["fmt"] == 8:
        x = x.view(torch.int8).float()
    else:
        x = torch.cat([x & 15, x >> 4], -2).float() - 8.0
    x = x * vs.float().unsqueeze(-2)
    return x.reshape(*vq.shape[:-2], -1, pt).transpose(-1, -2)


def _values16(s):
    """The whole pools of 8-bit codes as the values they stand for, f16: K [pages, H, NB, PT, 32], V [pages, H, NB, 32, PT]."""
    pages, kv, nb, pt = s["vs"].shape
    k = s["kq"].view(torch.int8) * s["ks"].transpose(2, 3).unsqueeze(-1)
    return k, s["vq"].view(torch.int8).view(pages, kv, nb, 32, pt) * s["vs"].unsqueeze(3)


def _softmax_parts(s):
    """Softmax weights [n, H, T, G] of every sequence's keys (zero past its length) and V [n, H, T, D]."""
    c = s["case"]
    nq, kv, d = _heads(c)
    n = c["seqs"]
    table = s["table"].long()
    keys = _k_values(c, s["kq"][table], s["ks"][table])                 # [n, pages, H, PT, D]
    keys = keys.transpose(1, 2).reshape(n, kv, -1, d)
    q = s["q"].float().view(n, kv, nq // kv, d).transpose(-1, -2).contiguous()
    sc = torch.matmul(keys, q) * s["scale"]                              # [n, H, T, G]
    del keys
    here = torch.arange(sc.shape[2], device=DEV)[None] < s["seq_len"][:, None]
    here = here[:, None, :, None]
    sc = torch.where(here, sc, -3.0e38)
    p = torch.where(here, torch.exp(sc - sc.amax(2, keepdim=True)), 0.0)
    p = p / torch.clamp(p.sum(2, keepdim=True), min=1e-30)
    values = _v_values(c, s["vq"][table], s["vs"][table])
    values = values.transpose(1, 2).reshape(n, kv, -1, d)
    return p, values


def _attend(s):
    c = s["case"]
    nq, _, d = _heads(c)
    p, values = _softmax_parts(s)
    o = torch.matmul(p.transpose(-1, -2).contiguous(), values)           # [n, H, G, D]
    return o.reshape(c["seqs"], nq, d).to(DTYPES[c["out"]]), p


def _run_evict(s):
    c = s["case"]
    _, kv, d = _heads(c)
    n, pt, nb, budget, longest = c["seqs"], c["pt"], d // 32, c["budget"], s["max_len"]
    lens = s["seq_len"].long()
    w = s["weights"]
    t = torch.arange(longest, device=DEV)[None]
    held = (t < c["sink"]) | (t >= lens[:, None] - c["recent"])
    rank = torch.where(w > 0, w, 0.0)
    rank = torch.where(held[:, None], math.inf, rank)
    rank = torch.where(t[:, None] < lens[:, None, None], rank, -1.0)
    order = torch.sort(rank, dim=-1, descending=True, stable=True)[1][..., :budget]
    n_kept = torch.clamp(lens, max=budget)
    i = torch.arange(order.shape[-1], device=DEV)
    order = torch.where(i < n_kept[:, None, None], order, longest)
    order = torch.sort(order, -1)[0]
    kept = torch.full((n, kv, budget), -1, dtype=torch.int32, device=DEV)
    kept[..., :order.shape[-1]] = torch.where(order < longest, order, -1).to(torch.int32)
    # the move: token kept[i] of a kv head to slot i of its new pages
    i = torch.arange(budget, device=DEV)
    live = (kept >= 0)
    src = torch.clamp(kept, min=0).long()
    rows = torch.arange(n, device=DEV)[:, None, None]
    h = torch.arange(kv, device=DEV)[None, :, None]
    page, slot = s["table"].long()[rows, src // pt], src % pt
    dpage, dslot = s["dst_table"].long()[:, None, i // pt].expand(n, kv, budget), (i % pt).expand(n, kv, budget)
    h = h.expand(n, kv, budget)
    for name in ("kq", "ks", "vq", "vs"):
        x = s[name] if name == "ks" else s[name].transpose(2, 3)         # [pages, H, PT, ..]
        new = torch.where(live[..., None] if x.dim() == 4 else live[..., None, None], x[page, h, slot], x[dpage, h, dslot])
        x[dpage, h, dslot] = new
    kept_w = torch.gather(w, 2, src)
    s["weights_out"].copy_(torch.where(live, kept_w, s["weights_out"]))
    return kept, n_kept.to(torch.int32), s["weights_out"], s["kq"], s["ks"], s["vq"], s["vs"]


def _inverse_frequencies(spec):
    """The rotated pairs' frequencies (64 bits) and the factor on cos and sin, by the usual scaling rules."""
    d, theta, f = spec["rotary_dim"], spec["theta"], spec["factor"]
    i = torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d
    if spec["scaling"] == "ntk":
        theta = theta * f ** (d / (d - 2))
    inv = theta ** -i
    if spec["scaling"] == "linear":
        return inv / f, 1.0
    if spec["scaling"] == "yarn":
        dim = lambda turns: d * math.log(spec["original_len"] / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(math.floor(dim(spec["high"])), 0), min(math.ceil(dim(spec["low"])), d - 1)
        ramp = torch.clamp((torch.arange(d // 2, device=DEV, dtype=torch.float64) - low) / max(high - low, 0.001), 0, 1)
        return inv / f * ramp + inv * (1 - ramp), 0.1 * math.log(f) + 1.0
    if spec["scaling"] == "bands":
        turns = spec["original_len"] * inv / (2 * math.pi)
        mix = torch.clamp((turns - spec["low"]) / (spec["high"] - spec["low"]), 0, 1)
        return inv / f * (1 - mix) + inv * mix, 1.0
    return inv, 1.0


def _rotate(s, x, weight):
    """Optional head RMSNorm, then the rotation, in 32 bits: x [n, new, heads, D]."""
    c = s["case"]
    inv, magnitude = _inverse_frequencies(s["spec"])
    angle = s["positions"].double()[..., None] * inv
    cos, sin = (torch.cos(angle) * magnitude).float()[:, :, None], (torch.sin(angle) * magnitude).float()[:, :, None]
    x = x.float()
    if c["normalise"]:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight
    r, rest = x[..., :c["rotary"]], x[..., c["rotary"]:]
    if c["layout"] == "half":
        a, b = r[..., :c["rotary"] // 2], r[..., c["rotary"] // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b = r[..., 0::2], r[..., 1::2]
    r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).reshape(r.shape)
    return torch.cat([r, rest], -1)


def _quantize(x):
    """Blocks of 32 along the last axis: int8 codes (halves away from zero) as bytes, and f16 scales."""
    d = x.abs().amax(-1, keepdim=True) / 127.0
    r = x * torch.where(d > 0, 1.0 / d, 0.0)
    codes = (torch.sign(r) * torch.floor(r.abs() + 0.5)).to(torch.int8).view(torch.uint8)
    return codes, d[..., 0].to(torch.float16)


def _run_append(s):
    c = s["case"]
    nq, kv, d = _heads(c)
    n, new, pt, nb = c["seqs"], c["new"], c["pt"], d // 32
    x = s["qkv"]
    q_out = _rotate(s, x[:, :, :nq], s["qw"]).to(DTYPES[c["out"]])
    k = _rotate(s, x[:, :, nq:nq + kv], s["kw"]).view(n, new, kv, nb, 32)
    v = x[:, :, nq + kv:].float().reshape(n, new, kv, nb, 32)
    at = s["start"].long()[:, None] + torch.arange(new, device=DEV)
    page = torch.gather(s["table"].long(), 1, at // pt)[..., None].expand(n, new, kv)
    slot = (at % pt)[..., None].expand(n, new, kv)
    h = torch.arange(kv, device=DEV).expand(n, new, kv)
    codes, scale = _quantize(k)
    s["kq"][page, h, :, slot] = codes
    s["ks"][page, h, slot] = scale
    codes, scale = _quantize(v)
    s["vq"][page, h, :, slot] = codes.reshape(n, new, kv, -1)
    s["vs"][page, h, :, slot] = scale
    return (q_out,) + _values16(s)


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    if c["op"] == "shared":
        return _attend(s)[0]
    if c["op"] == "weights":
        out, p = _attend(s)
        here = torch.arange(s["max_len"], device=DEV) < s["seq_len"][:, None, None]  # the rest of a row is left as it is
        s["weights_out"].copy_(torch.where(here, s["weights"] + p.sum(-1)[..., :s["max_len"]], s["weights_out"]))
        return out, s["weights_out"]
    if c["op"] == "evict":
        return _run_evict(s)
    if c["op"] == "rotary":
        nq, kv, _ = _heads(c)
        x = s["qkv"]
        return (_rotate(s, x[:, :, :nq], s["qw"]).to(DTYPES[c["out"]]),
                _rotate(s, x[:, :, nq:nq + kv], s["kw"]).to(DTYPES[c["out"]]))
    return _run_append(s)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------

def work(case):
    nq, kv, d = _heads(case)
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] in ("rotary", "append"):
        tokens = case["seqs"] * case["new"]
        rows = tokens * (nq + kv) * d
        b = rows * size[case["src"]] + rows * size[case["out"]]
        if case["op"] == "append":
            per = kv * d // 32 * ((32 if case["fmt"] == 8 else 16) + 2)
            b += tokens * (kv * d * (size[case["src"]] - size[case["out"]]) + 2 * per)
        return {"bytes": float(b), "flops": float(rows * 4)}
    per = 2 * kv * (d // 32) * ((32 if case["fmt"] == 8 else 16) + 2)  # K and V of one token
    n = case["seqs"]
    if case["op"] == "shared":  # prefixes once each, half the longest tail on average
        keys = case["prefix"] * (1 + 0.75 * (case["groups"] - 1)) + n * case["tail"] / 2
        seen = n * (case["prefix"] * (1 if case["groups"] == 1 else 0.8) + case["tail"] / 2)
        return {"bytes": keys * per + n * nq * d * (size[case["q"]] + size[case["out"]]), "flops": 4.0 * seen * nq * d}
    keys = case["longest"] * (1 + 0.5 * (n - 1))  # the lengths are spread over the whole range
    if case["op"] == "weights":
        return {"bytes": keys * (per + 8 * kv) + n * nq * d * (size[case["q"]] + size[case["out"]]),
                "flops": 4.0 * keys * nq * d}
    moved = min(case["budget"], case["longest"]) * (1 + 0.75 * (n - 1))
    return {"bytes": keys * kv * 4 + moved * (2 * per + kv * 12), "flops": keys * kv}


# ---- the definitions, in 64 bits, one sequence at a time ----------------------------------------------------------------------

def _exact_cache(s, i):
    """K and V of sequence i as float64 [T, H, D]: value = scale * code, read off the documented layout."""
    c = s["case"]
    _, kv, d = _heads(c)
    pt, nb, t = c["pt"], d // 32, int(s["seq_len"][i])
    pages = s["table"][i, :-(-t // pt)].long()
    kq, ks, vq, vs = (s[x][pages] for x in ("kq", "ks", "vq", "vs"))
    if c["fmt"] == 8:
        k = kq.view(torch.int8).double().permute(0, 3, 1, 2, 4)                          # [page, slot, H, NB, 32]
        v = vq.view(torch.int8).double().view(-1, kv, nb, 32, pt).permute(0, 4, 1, 2, 3)
    else:
        low, high = (kq % 16).double() - 8, torch.div(kq, 16, rounding_mode="floor").double() - 8
        k = torch.stack([low, high], -2).flatten(-2).permute(0, 3, 1, 2, 4)
        x = vq.view(-1, kv, nb, 16, pt)
        low, high = (x % 16).double() - 8, torch.div(x, 16, rounding_mode="floor").double() - 8
        v = torch.stack([low, high], 3).flatten(3, 4).permute(0, 4, 1, 2, 3)
    k = k * ks.double().permute(0, 2, 1, 3)[..., None]
    v = v * vs.double().permute(0, 3, 1, 2)[..., None]
    return k.reshape(-1, kv, d)[:t], v.reshape(-1, kv, d)[:t]


def _exact_attend(s):
    c = s["case"]
    nq, kv, d = _heads(c)
    out = torch.zeros(c["seqs"], nq, d, dtype=torch.float64, device=DEV)
    weight = torch.zeros(c["seqs"], kv, s["max_len"], dtype=torch.float64, device=DEV)
    for i in range(c["seqs"]):
        t = int(s["seq_len"][i])
        if t == 0:
            continue
        k, v = _exact_cache(s, i)
        for h in range(kv):
            rows = slice(h * (nq // kv), (h + 1) * (nq // kv))
            p = torch.softmax(s["q"][i, rows].double() @ k[:, h].t().contiguous() * s["scale"], -1)
            out[i, rows] = p @ v[:, h].contiguous()
            weight[i, h, :t] = p.sum(0)
    return out, weight


def _exact_frequencies(spec):
    half = spec["rotary_dim"] // 2
    f, length, base = spec["factor"], spec["original_len"], spec["theta"]
    if spec["scaling"] == "ntk":
        base *= f ** (2 * half / (2 * half - 2))
    inv = np.array([base ** (-j / half) for j in range(half)])
    if spec["scaling"] == "linear":
        return inv / f, 1.0
    if spec["scaling"] == "yarn":
        edge = [half * math.log(length / (2 * math.pi * turns)) / math.log(base) for turns in (spec["high"], spec["low"])]
        low, high = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), 2 * half - 1)
        share = np.array([min(1.0, max(0.0, (j - low) / max(high - low, 0.001))) for j in range(half)])
        return inv * (1 - share) + inv * share / f, 1 + 0.1 * math.log(f)
    if spec["scaling"] == "bands":
        got = []
        for w in inv:
            wave = 2 * math.pi / w
            if wave < length / spec["high"]:
                got.append(w)
            elif wave > length / spec["low"]:
                got.append(w / f)
            else:
                m = (length / wave - spec["low"]) / (spec["high"] - spec["low"])
                got.append((1 - m) * w / f + m * w)
        return np.array(got), 1.0
    return inv, 1.0


def _exact_rotate(s, x, weight):
    c = s["case"]
    inv, magnitude = _exact_frequencies(s["spec"])
    x = x.double()
    if c["normalise"]:
        x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * weight.double()
    angle = s["positions"].double()[..., None, None] * torch.from_numpy(inv).to(DEV)
    z = magnitude * torch.polar(torch.ones_like(angle), angle)
    r = c["rotary"]
    first, second = (x[..., :r // 2], x[..., r // 2:r]) if c["layout"] == "half" else (x[..., 0:r:2], x[..., 1:r:2])
    z = torch.complex(first.contiguous(), second.contiguous()) * z
    out = x.clone()
    if c["layout"] == "half":
        out[..., :r // 2], out[..., r // 2:r] = z.real, z.imag
    else:
        out[..., 0:r:2], out[..., 1:r:2] = z.real, z.imag
    return out


def _exact_quantized(x):
    """float64 [.., NB, 32] as the values its stored 8-bit codes and f16 scale stand for."""
    d = x.abs().amax(-1, keepdim=True) / 127
    some = d > 0
    r = x / torch.where(some, d, 1.0)
    return torch.where(some, torch.trunc(r + torch.copysign(torch.full_like(x, 0.5), x)), 0.0) * d.to(torch.float16).double()


def exact(case, seed):
    s = prepare(case, seed)
    nq, kv, d = _heads(case)
    if case["op"] == "shared":
        return _exact_attend(s)[0]
    if case["op"] == "weights":
        out, w = _exact_attend(s)
        here = torch.arange(s["max_len"], device=DEV) < s["seq_len"][:, None, None]
        return out, torch.where(here, w + s["weights"].double(), s["weights_out"].double())
    if case["op"] == "evict":
        return None  # whole numbers and moved values: nothing is computed
    x = s["qkv"]
    q = _exact_rotate(s, x[:, :, :nq], s["qw"])
    k = _exact_rotate(s, x[:, :, nq:nq + kv], s["kw"])
    if case["op"] == "rotary":
        return q, k
    n, new, pt, nb = case["seqs"], case["new"], case["pt"], d // 32
    kval, vval = (t.double() for t in _values16(s))
    kn = _exact_quantized(k.view(n, new, kv, nb, 32))
    vn = _exact_quantized(x[:, :, nq + kv:].double().reshape(n, new, kv, nb, 32))
    table, start = s["table"].cpu().numpy(), s["start"].cpu().numpy()
    for i in range(n):
        pos = start[i] + np.arange(new)
        page, slot = torch.from_numpy(table[i][pos // pt]).long().to(DEV), torch.from_numpy(pos % pt).long().to(DEV)
        kval[page, :, :, slot] = kn[i]
        vval[page, :, :, :, slot] = vn[i]
    return q, kval, vval
