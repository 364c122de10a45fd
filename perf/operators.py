"""Cases for the text-side operators: rotary positions, masked / capped / biased attention, and
attention of a batch that shares a prefix.

``run`` computes them in elementary torch operations (32 bits, angles in 64), or through
quantfun2_b200 where ``own`` is true.  ``exact`` is the definition in 64 bits.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------- cases --
def _rotary(name, **kw):
    c = dict(name=name, op="rotary", dtype="bf16", batch=1, length=1, heads=24, kv_heads=8, dim=128, rotary=128,
             layout="half", scaling="none", factor=1.0, farthest=8192)
    c.update(kw)
    return c


def _attention(name, **kw):
    c = dict(name=name, op="attention", dtype="bf16", batch=1, heads=24, kv_heads=8, dim=128, q_len=1, kv_len=1,
             causal=False, left=-1, prefix=0, documents=0, padded=False, ragged=False, cap=0.0, bias="none", reach=0,
             scale=0.0, shared=0, geometry=1)
    c.update(kw)
    return c


def listed():
    return [
        # one decoding step of a batch: every head of one token each, far into a long context
        _rotary("rotary single tokens", batch=16, length=1, scaling="by_parts", factor=8.0, farthest=131072),
        # a batch of prompts, a part of each head rotated in interleaved pairs, fp16
        _rotary("rotary partial prompts", dtype="fp16", batch=4, length=1021, heads=16, kv_heads=16, dim=96, rotary=32,
                layout="interleaved", farthest=4096),
        # a long document in one pass
        _rotary("rotary long", batch=1, length=65537, scaling="linear", factor=4.0, farthest=131072),
        # the shortest text: a causal encoder's prompt window
        _attention("causal prompts", dtype="fp16", batch=2, heads=12, kv_heads=12, dim=64, q_len=77, kv_len=77,
                   causal=True),
        # padded prompts in a causal sliding window with capped scores, wide heads
        _attention("capped window", batch=4, heads=8, kv_heads=4, dim=256, q_len=1000, kv_len=1000, causal=True,
                   left=511, padded=True, cap=50.0),
        # a bidirectional encoder with a learned bias by distance, unscaled scores, padded prompts
        _attention("distance table", batch=4, heads=64, kv_heads=64, dim=64, q_len=512, kv_len=512, padded=True,
                   bias="table", reach=128, scale=1.0),
        # many texts packed into one sequence
        _attention("documents", batch=1, dim=96, q_len=16384, kv_len=16384, documents=24),
        # a text prefix that all see, and causal tokens after it
        _attention("prefix", batch=2, dim=96, q_len=4352, kv_len=4352, causal=True, prefix=256),
        # a long causal pass: the largest
        _attention("long causal", q_len=16384, kv_len=16384, causal=True),
        # single tokens on long caches of unlike lengths, linear bias by distance
        _attention("single tokens", batch=4, q_len=1, kv_len=32768, causal=True, ragged=True, bias="slopes"),
        # prompts behind one system text
        _attention("shared prompts", op="shared", batch=16, q_len=256, kv_len=256, causal=True, ragged=True,
                   shared=1000),
        # single tokens of many answers behind one long text
        _attention("shared single tokens", op="shared", batch=64, q_len=1, kv_len=512, causal=True, ragged=True,
                   shared=16384),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotary", "attention", "attention", "single", "shared", "shared single"])
    if kind == "rotary":
        dim = rng.choice([64, 96, 128, 256])
        kv = rng.choice([1, 4, 8, 12])
        c = _rotary("", dtype=rng.choice(["bf16", "fp16", "fp32"]), batch=rng.randint(1, 16), heads=kv * rng.randint(1, 4),
                    kv_heads=kv, dim=dim, rotary=rng.choice([dim, dim // 2, dim // 4]),
                    layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "by_parts"]),
                    factor=rng.choice([2.0, 4.0, 8.0]), farthest=_log_int(rng, 1000, 1000000))
        # at most the elements of the longest listed case
        most = 65537 * 32 * 128 // (2 * c["batch"] * (c["heads"] + kv) * dim)
        c["length"] = _log_int(rng, 1, max(2, min(65537, most)))
    else:
        kv = rng.choice([1, 2, 4, 8, 12])
        group = rng.choice([1, 1, 2, 3, 4])
        dim = rng.choice([64, 96, 128, 256])
        c = _attention("", dtype=rng.choice(["bf16", "fp16"]), heads=kv * group, kv_heads=kv, dim=dim,
                       cap=rng.choice([0.0, 0.0, 30.0, 50.0]), bias=rng.choice(["none", "none", "slopes", "table"]),
                       geometry=rng.randint(1, 1 << 30))
        if c["bias"] == "table":
            c["reach"] = rng.choice([32, 128, 500])
        if kind == "attention":
            c["batch"] = rng.randint(1, 4)
            # at most the products of the longest listed case, were every pair seen
            most = int(math.sqrt(1.6e12 / (4 * dim * c["heads"] * c["batch"])))
            n = _log_int(rng, 33, min(8000, most))
            c.update(q_len=n, kv_len=n, causal=rng.random() < 0.6)
            mask = rng.choice(["none", "window", "prefix", "documents", "padded"])
            if mask == "window":
                c["left"] = rng.randint(0, n)
            elif mask == "prefix":
                c.update(causal=True, prefix=rng.randint(1, n))
            elif mask == "documents":
                c["documents"] = rng.randint(2, 20)
            elif mask == "padded":
                c["padded"] = True
        elif kind == "single":
            c["batch"] = _log_int(rng, 1, 16)
            most = int(1.0e9 / (4 * dim * kv * c["batch"]))
            c.update(q_len=rng.choice([1, 1, 1, 2, 5]), kv_len=_log_int(rng, 100, min(30000, most)), causal=True,
                     ragged=True)
            if rng.random() < 0.3:
                c["left"] = rng.randint(1, c["kv_len"])
        elif kind == "shared":
            n = rng.randint(20, 400)
            c.update(op="shared", batch=rng.randint(2, 16), q_len=n, kv_len=n, causal=True, ragged=True,
                     shared=_log_int(rng, 50, 4000))
        else:
            c.update(op="shared", batch=rng.randint(2, 64), q_len=1, kv_len=rng.randint(1, 600), causal=True, ragged=True,
                     shared=_log_int(rng, 500, 16384))
    del c["name"]
    return c


# ---------------------------------------------------------------- geometry --
def _geometry(case):
    """Lengths, offsets, prefixes and document ids of an attention case, from the case alone
    (numpy; positions count the shared prefix)."""
    rng = random.Random(case["geometry"])
    B, Sq, Skv, P = case["batch"], case["q_len"], case["kv_len"], case["shared"]
    lens = [Skv] * B
    if case["ragged"]:
        least = max(1, Skv // 2) if Sq == Skv else max(Sq, Skv // 2)
        lens = [rng.randint(least, Skv) for _ in range(B)]
    # a prompt's queries are its keys' tokens; fewer queries than keys are the last ones
    offsets = [0 if Sq == Skv else n - Sq for n in lens]
    prefix = [rng.randint(1, case["prefix"]) if case["prefix"] else 0 for _ in range(B)]
    ids = None
    if case["documents"]:
        ids = np.zeros((B, Skv), np.int32)
        for b in range(B):
            cuts = sorted(rng.randint(0, Skv) for _ in range(case["documents"] - 1))
            for cut in cuts:
                ids[b, cut:] += 1
    elif case["padded"]:
        ids = np.zeros((B, Skv), np.int32)
        for b in range(B):
            ids[b, rng.randint(Skv // 4, Skv):] = -1
    return dict(lens=np.array(lens, np.int32), offsets=np.array(offsets, np.int32), prefix=np.array(prefix, np.int32),
                ids=ids, shared=P)


def _pairs(case):
    """Pairs of query and key that are seen, of one query head, and tokens that take part."""
    g = _geometry(case)
    B, Sq, Skv, P = case["batch"], case["q_len"], case["kv_len"], case["shared"]
    pairs = rows = 0
    keys = P
    for b in range(B):
        t = P + g["offsets"][b] + np.arange(Sq, dtype=np.int64)
        n = P + int(g["lens"][b])
        lo = np.maximum(t - case["left"], 0) if case["left"] >= 0 else np.zeros_like(t)
        hi = np.minimum(t + 1, n) if case["causal"] else np.full_like(t, n)
        pre = np.full_like(t, min(int(g["prefix"][b]), n))
        live = np.ones(Sq, bool)
        if g["ids"] is not None:
            own_id = g["ids"][b][t]
            live = own_id >= 0
            first = np.searchsorted(np.where(g["ids"][b] < 0, 1 << 30, g["ids"][b]), own_id, "left")
            last = np.searchsorted(np.where(g["ids"][b] < 0, 1 << 30, g["ids"][b]), own_id, "right")
            lo, hi = np.maximum(lo, first), np.minimum(hi, last)
            keys += int((g["ids"][b] >= 0).sum())
        else:
            # single tokens in a window need the window's keys alone
            keys += n - P if not (case["left"] >= 0 and Sq < Skv) else int(min(n - P, case["left"] + Sq))
        band = np.maximum(hi - lo, 0)
        more = np.maximum(pre - np.maximum(hi, 0), 0) + np.minimum(np.maximum(lo, 0), pre)
        pairs += int(((band + np.where(pre > 0, more, 0)) * live).sum())
        rows += int(live.sum())
    return pairs, rows, keys


def work(case):
    if case["op"] == "rotary":
        size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
        tokens, heads = case["batch"] * case["length"], case["heads"] + case["kv_heads"]
        return {"bytes": 2 * tokens * heads * case["dim"] * size + 8 * tokens,
                "flops": 3 * tokens * heads * case["rotary"]}
    pairs, rows, keys = _pairs(case)
    out_rows = case["batch"] * case["q_len"]
    return {"bytes": 2 * case["dim"] * (case["heads"] * (rows + out_rows) + 2 * case["kv_heads"] * keys),
            "flops": 4 * case["dim"] * case["heads"] * pairs}


# ------------------------------------------------------------------ inputs --
def _inv_freq(case):
    """Frequencies of the rotated pairs, 64 bits: base 10000, stretched for long contexts."""
    r = case["rotary"]
    f = 10000.0 ** (-np.arange(0, r, 2, dtype=np.float64) / r)
    if case["scaling"] == "linear":
        f = f / case["factor"]
    elif case["scaling"] == "by_parts":
        # pairs that turn often over the first length are kept, slow ones are stretched
        first, fast, slow = 4096.0, 32.0, 1.0
        turns = first * f / (2 * math.pi)
        keep = np.clip((turns - slow) / (fast - slow), 0.0, 1.0)
        f = f * keep + f / case["factor"] * (1 - keep)
    return f


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    randn = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    B, H, Hk, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    st = {"case": case}
    if case["op"] == "rotary":
        S = case["length"]
        st["q"], st["k"] = randn(B, S, H, D).to(dt), randn(B, S, Hk, D).to(dt)
        far = max(1, case["farthest"] - S)
        start = torch.randint(0, far, (B, 1), device=dev, generator=g)
        st["positions"] = start + torch.arange(S, device=dev)[None]
        st["inv_freq"] = torch.from_numpy(_inv_freq(case)).to(dev)
        st["magnitude"] = 1.0 if case["scaling"] != "by_parts" else 0.1 * math.log(case["factor"]) + 1.0
        return st
    Sq, Skv, P = case["q_len"], case["kv_len"], case["shared"]
    # normalised heads: unit variance, some directions of the keys shared by all tokens; unscaled scores come
    # with small queries
    wide = case["scale"] or 1.0 / math.sqrt(D)
    q = randn(B, Sq, H, D) * (1.5 if not case["scale"] else 1.0 / math.sqrt(D))
    st["q"] = q.to(dt)
    common = randn(1, 1, Hk, D) * 0.5
    st["k"], st["v"] = (randn(B, Skv, Hk, D) + common).to(dt), randn(B, Skv, Hk, D).to(dt)
    if P:
        st["prefix_k"], st["prefix_v"] = (randn(P, Hk, D) + common[0]).to(dt), randn(P, Hk, D).to(dt)
    geo = _geometry(case)
    st["scale"] = wide
    st["lens"] = torch.from_numpy(geo["lens"]).to(dev) if case["ragged"] else None
    st["prefix_lens"] = torch.from_numpy(geo["prefix"]).to(dev) if case["prefix"] else None
    st["ids"] = torch.from_numpy(geo["ids"]).to(dev) if geo["ids"] is not None else None
    st["offsets"] = torch.from_numpy(geo["offsets"]).to(dev)
    st["slopes"] = st["table"] = None
    if case["bias"] == "slopes":
        st["slopes"] = torch.exp2(-8.0 * torch.arange(1, H + 1, device=dev, dtype=torch.float32) / H)
    elif case["bias"] == "table":
        st["table"] = randn(H, 2 * case["reach"] + 1)
    return st


# --------------------------------------------------------------- own calls --
def _run_own(st):
    from quantfun2_b200 import attention, kernels

    c = st["case"]
    if c["op"] == "rotary":
        return kernels.rotary_apply(st["q"], st["k"], st["positions"], st["inv_freq"], layout=c["layout"],
                                    magnitude=st["magnitude"])
    window = (c["left"], 0 if c["causal"] else -1)
    # fewer queries than keys are the last tokens of each sequence
    offset = 0 if c["q_len"] == c["kv_len"] else "end"
    more = dict(window=window, kv_lens=st["lens"], q_offset=offset, softcap=c["cap"], slopes=st["slopes"],
                bias_table=st["table"], sm_scale=st["scale"], tensor_layout="NHD")
    if c["op"] == "shared":
        return attention.shared_prefix_attn(st["q"], st["prefix_k"], st["prefix_v"], st["k"], st["v"], **more)
    return attention.masked_attn(st["q"], st["k"], st["v"], prefix_lens=st["prefix_lens"], segment_ids=st["ids"], **more)


# -------------------------------------------------------------- plain form --
def _run_rotary(st):
    c = st["case"]
    r, half = c["rotary"], c["rotary"] // 2
    angle = st["positions"].double()[..., None] * st["inv_freq"]
    cos = (angle.cos() * st["magnitude"]).float()[:, :, None]
    sin = (angle.sin() * st["magnitude"]).float()[:, :, None]
    outs = []
    for x in (st["q"], st["k"]):
        y = x.float()
        rot, rest = y[..., :r], y[..., r:]
        if c["layout"] == "half":
            a, b = rot[..., :half], rot[..., half:]
            rot = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = rot[..., 0::2], rot[..., 1::2]
            rot = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        outs.append(torch.cat([rot, rest], -1).to(x.dtype))
    return tuple(outs)


def _seen(c, st, b, t, pos):
    """[rows, keys] truth values: does the query at position t see the key at pos (batch element b)."""
    P = c["shared"]
    n = P + (st["lens"][b] if st["lens"] is not None else c["kv_len"])
    d = pos[None, :] - t[:, None]
    band = torch.ones_like(d, dtype=torch.bool)
    if c["causal"]:
        band &= d <= 0
    if c["left"] >= 0:
        band &= d >= -c["left"]
    if st["prefix_lens"] is not None:
        band |= (pos < st["prefix_lens"][b])[None, :]
    band &= (pos < n)[None, :]
    if st["ids"] is not None:
        qi, ki = st["ids"][b][t], st["ids"][b][pos]
        band &= (qi[:, None] == ki[None, :]) & (qi >= 0)[:, None]
    return band, d


def _run_attention(st):
    c = st["case"]
    H, Hk, D, P = c["heads"], c["kv_heads"], c["dim"], c["shared"]
    G = H // Hk
    dev = st["q"].device
    out = torch.empty_like(st["q"])
    pos = torch.arange(P + c["kv_len"], device=dev)
    # score rows at a time so that a chunk stays near 2^28 elements
    rows = max(1, min(c["q_len"], (1 << 28) // max(1, H * pos.numel())))
    for b in range(c["batch"]):
        k, v = st["k"][b].float(), st["v"][b].float()
        if P:
            k, v = torch.cat([st["prefix_k"].float(), k]), torch.cat([st["prefix_v"].float(), v])
        k, v = k.transpose(0, 1), v.transpose(0, 1)                               # [Hk, keys, D]
        if c["ragged"]:
            v = torch.where((pos < P + st["lens"][b])[None, :, None], v, 0.0)
        for r0 in range(0, c["q_len"], rows):
            q = st["q"][b, r0:r0 + rows].float()                                   # [rows, H, D]
            n = q.shape[0]
            t = P + st["offsets"][b] + torch.arange(r0, r0 + n, device=dev)
            seen, d = _seen(c, st, b, t, pos)
            q = q.view(n, Hk, G, D).permute(1, 2, 0, 3).reshape(Hk, G * n, D)
            s = torch.matmul(q, k.transpose(1, 2)).view(H, n, -1) * st["scale"]
            if c["cap"] > 0:
                s = c["cap"] * torch.tanh(s / c["cap"])
            if st["slopes"] is not None:
                s = s - st["slopes"][:, None, None] * d.abs()
            if st["table"] is not None:
                s = s + st["table"][:, d.clamp(-c["reach"], c["reach"]) + c["reach"]]
            s = s.masked_fill(~seen, -math.inf)
            m = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(torch.isinf(m), 0.0, m))
            z = p.sum(-1, keepdim=True)
            o = torch.matmul(p.view(Hk, G * n, -1), v).view(H, n, D) / torch.where(z > 0, z, 1.0)
            out[b, r0:r0 + n] = o.transpose(0, 1).to(out.dtype)
    return out


def run(state):
    if own:
        return _run_own(state)
    return _run_rotary(state) if state["case"]["op"] == "rotary" else _run_attention(state)


# ------------------------------------------------------------------- exact --
def exact(case, seed):
    st = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "rotary":
        r = case["rotary"]
        z = torch.polar(torch.full_like(st["inv_freq"], st["magnitude"]).expand(*st["positions"].shape, r // 2),
                        st["positions"].to(f64).unsqueeze(-1) * st["inv_freq"]).unsqueeze(2)
        res = []
        for x in (st["q"], st["k"]):
            y = x.to(f64)
            pairs = y[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2) if case["layout"] == "half" else \
                y[..., :r].unflatten(-1, (r // 2, 2))
            w = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
            y[..., :r] = (w.transpose(-1, -2) if case["layout"] == "half" else w).flatten(-2)
            res.append(y)
        return tuple(res)
    B, H, D, P = case["batch"], case["heads"], case["dim"], case["shared"]
    G = H // case["kv_heads"]
    pairs, _, _ = _pairs(case)
    total = P + case["kv_len"]
    if B * H * case["q_len"] * total > 2.0e10:
        return None
    geo = _geometry(case)
    dev = st["q"].device
    out = torch.zeros(B, case["q_len"], H, D, dtype=f64, device=dev)
    j = torch.arange(total, device=dev)
    step = max(1, (1 << 26) // total)
    for b in range(B):
        n = P + int(geo["lens"][b])
        pre = int(geo["prefix"][b])
        for r0 in range(0, case["q_len"], step):
            i = torch.arange(r0, min(case["q_len"], r0 + step), device=dev)
            t = P + int(geo["offsets"][b]) + i
            # the keys that any of these rows can see
            lo = max(0, int(t[0]) - case["left"]) if case["left"] >= 0 and not pre else 0
            hi = max(min(n, int(t[-1]) + 1), min(n, pre)) if case["causal"] else n
            jj = j[lo:hi]
            ok = torch.ones(i.numel(), jj.numel(), dtype=torch.bool, device=dev)
            if case["left"] >= 0:
                ok &= t[:, None] - jj <= case["left"]
            if case["causal"]:
                ok &= t[:, None] >= jj
            ok |= jj < pre
            if geo["ids"] is not None:
                ids = st["ids"][b]
                ok &= (ids[t][:, None] == ids[jj]) & (ids[jj] >= 0)
            gone = ~ok.any(1)
            for h in range(H):
                kk, vv = st["k"][b, :, h // G].to(f64), st["v"][b, :, h // G].to(f64)
                if P:
                    kk = torch.cat([st["prefix_k"][:, h // G].to(f64), kk])
                    vv = torch.cat([st["prefix_v"][:, h // G].to(f64), vv])
                s = st["q"][b, i, h].to(f64) @ kk[jj].T * st["scale"]
                if case["cap"] > 0:
                    s = torch.tanh(s / case["cap"]) * case["cap"]
                if case["bias"] == "slopes":
                    s = s - st["slopes"][h].to(f64) * (t[:, None] - jj).abs()
                if case["bias"] == "table":
                    s = s + st["table"][h].to(f64)[(jj - t[:, None]).clamp(-case["reach"], case["reach"]) + case["reach"]]
                s = torch.where(ok, s, torch.full((), -math.inf, dtype=f64, device=dev))
                s[gone] = 0.0
                p = torch.softmax(s, -1)
                p[gone] = 0.0
                out[b, i, h] = p @ vv[jj]
    return out
