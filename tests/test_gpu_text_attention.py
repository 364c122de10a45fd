"""GPU: masked, capped and biased attention and its shared-prefix form against the 64-bit
formula (oracle.text), with the elementwise bound derived there."""
import math

import pytest
import torch

from oracle import text as ot

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def _inputs(dev, B, Sq, Skv, Hq, Hkv, D, dtype, seed=0, P=0, amp=1.5):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    q = (r(B, Sq, Hq, D) * amp).to(dtype)
    k = (r(B, Skv, Hkv, D) + 0.5 * r(1, 1, Hkv, D)).to(dtype)
    v = r(B, Skv, Hkv, D).to(dtype)
    if P:
        return q, k, v, r(P, Hkv, D).to(dtype), r(P, Hkv, D).to(dtype)
    return q, k, v


def _compare(out, q, k, v, offsets=None, kv_lens=None, rows=None, **kw):
    """out against the oracle on all rows, or on the listed ones."""
    from quantfun2_b200 import attention as A

    A.masked_attn_status()
    Sq, Skv = q.shape[1], k.shape[1]
    if rows is not None:
        base = [Skv - Sq if offsets is None else int(offsets[b]) for b in range(q.shape[0])]
        refs = []
        for i in rows:
            sub = dict(kw)
            if kw.get("q_ids") is not None:
                sub["q_ids"] = kw["q_ids"][:, i:i + 1]
            refs.append(ot.attention(q[:, i:i + 1], k, v, offsets=[o + i for o in base], kv_lens=kv_lens, **sub))
        ref, mag, keys = (torch.cat([r[n] for r in refs], 1) for n in range(3))
        out = out[:, rows]
    else:
        ref, mag, keys = ot.attention(q, k, v, offsets=offsets, kv_lens=kv_lens, **kw)
    v_max = v[torch.isfinite(v)].abs().max().double().item() if v.numel() else 0.0
    if kw.get("prefix_v") is not None:
        v_max = max(v_max, kw["prefix_v"].abs().max().double().item())
    tol = ot.attention_bound(ref, mag, keys, q.dtype, v_max)
    err = (out.double() - ref).abs()
    assert torch.isfinite(out).all()
    assert (err <= tol).all(), f"{(err / tol).max().item():.3f} of the bound, {err.max().item():.4g} off"
    assert not out[(keys == 0)].any()


def _window(causal, left=-1):
    return (left, 0 if causal else -1)


# lengths around the tile edges, head dims, groups, both directions, both types
@pytest.mark.parametrize("B,Sq,Hq,Hkv,D,dtype,causal", [
    (1, 1, 1, 1, 64, BF16, True), (2, 1, 3, 1, 128, FP16, False), (1, 2, 4, 2, 96, BF16, True),
    (2, 77, 4, 4, 64, FP16, True), (1, 127, 2, 2, 128, BF16, True), (1, 128, 3, 1, 256, BF16, True),
    (1, 129, 2, 1, 64, BF16, False), (2, 200, 4, 1, 256, FP16, True), (1, 257, 6, 2, 96, FP16, True),
    (1, 300, 2, 2, 128, FP16, False), (1, 385, 5, 5, 128, BF16, True), (1, 33, 40, 1, 128, BF16, True),
    (1, 3, 130, 1, 64, BF16, True),
])
def test_dense_and_causal(cuda, B, Sq, Hq, Hkv, D, dtype, causal):
    from quantfun2_b200 import attention as A

    q, k, v = _inputs(cuda, B, Sq, Sq, Hq, Hkv, D, dtype, seed=Sq)
    out = A.masked_attn(q, k, v, window=_window(causal), tensor_layout="NHD")
    _compare(out, q, k, v, window=_window(causal))
    hnd = A.masked_attn(q.transpose(1, 2).contiguous(), k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous(),
                        window=_window(causal))
    assert torch.equal(hnd.transpose(1, 2), out)


# grids that fill the SMs (heads * batch large), spot rows
@pytest.mark.parametrize("B,S,Hq,Hkv,D,dtype,window", [
    (4, 300, 40, 8, 64, BF16, (-1, 0)), (3, 513, 24, 8, 96, FP16, (-1, -1)), (8, 640, 24, 24, 128, BF16, (100, 0)),
    (4, 1000, 24, 8, 128, BF16, (-1, 0)), (2, 1281, 24, 8, 128, FP16, (130, 40)), (13, 257, 12, 12, 64, FP16, (0, 0)),
])
def test_two_tile_grids(cuda, B, S, Hq, Hkv, D, dtype, window):
    from quantfun2_b200 import attention as A

    q, k, v = _inputs(cuda, B, S, S, Hq, Hkv, D, dtype, seed=S)
    out = A.masked_attn(q, k, v, window=window, tensor_layout="NHD")
    rows = sorted({0, 1, 31, 127, 128, 129, 255, 256, S // 2, S - 2, S - 1})
    _compare(out, q, k, v, rows=rows, window=window)


# Long key ranges and grids that fill the SMs: two query tiles in one CTA (short ranges, as in the
# tests above, are taken by CTAs of one tile).
PAIR_ROWS = [0, 1, 31, 127, 128, 129, 255, 256]


@pytest.mark.parametrize("B,Sq,Skv,Hq,Hkv,D,dtype,window", [
    (4, 390, 2600, 24, 8, 64, BF16, (-1, 0)), (4, 511, 2561, 24, 24, 96, FP16, (-1, -1)), (4, 512, 2688, 24, 8, 128, BF16, (1700, 0)),
    (1, 2305, 2305, 18, 6, 128, FP16, (-1, -1)), (8, 450, 5000, 24, 8, 128, BF16, (-1, 300)), (2, 600, 3001, 48, 1, 96, BF16, (2200, 40)),
])
def test_pairs_of_query_tiles(cuda, B, Sq, Skv, Hq, Hkv, D, dtype, window):
    from quantfun2_b200 import attention as A

    q, k, v = _inputs(cuda, B, Sq, Skv, Hq, Hkv, D, dtype, seed=Sq)
    buf = torch.full((B, Sq + 3, Hq + 1, D), 3.0, device=cuda, dtype=dtype)
    out = A.masked_attn(q, k, v, window=window, tensor_layout="NHD", out=buf[:, 1:Sq + 1, 1:])
    rows = sorted({*PAIR_ROWS, Sq // 2, Sq - 2, Sq - 1})
    _compare(out, q, k, v, rows=rows, window=window)
    assert torch.equal(out, A.masked_attn(q, k, v, window=window, tensor_layout="NHD"))
    buf[:, 1:Sq + 1, 1:] = 3.0
    assert (buf == 3.0).all()                              # nothing beside the view was written


@pytest.mark.parametrize("D,dtype", [(64, FP16), (96, BF16), (128, BF16)])
def test_pairs_with_capped_and_biased_scores(cuda, D, dtype):
    from quantfun2_b200 import attention as A

    B, Sq, Skv, Hq = 3, 500, 2500, 32
    q, k, v = _inputs(cuda, B, Sq, Skv, Hq, Hq // 2, D, dtype, seed=6, amp=4.0)
    slopes = torch.rand(Hq, device=cuda) * 0.2
    rows = [0, 127, 128, 300, 499]
    calls = [dict(bias_table=torch.randn(Hq, 2 * R + 1, device=cuda)) for R in (0, 40, 1024)]
    calls += [dict(softcap=2.0, window=(-1, 0)), dict(softcap=50.0), dict(slopes=slopes), dict(slopes=slopes, window=(-1, 0)),
              dict(softcap=50.0, slopes=slopes, window=(2100, 20), sm_scale=0.3)]
    for kw in calls:
        out = A.masked_attn(q, k, v, tensor_layout="NHD", **kw)
        _compare(out, q, k, v, rows=rows, **kw)


def test_pairs_with_prefixes_lengths_and_documents(cuda):
    from quantfun2_b200 import attention as A

    B, S, Hq, Hkv, D = 5, 500, 24, 8, 96
    Skv = 2500
    q, k, v = _inputs(cuda, B, S, Skv, Hq, Hkv, D, BF16, seed=7)
    pre = torch.tensor([0, 1, 128, 1500, 9999], device=cuda)
    lens = torch.tensor([2500, 0, 1, 129, 5000], device=cuda, dtype=torch.int32)
    off = torch.tensor([2000, 0, -600, 50, 1], device=cuda, dtype=torch.int32)
    rows = [0, 127, 128, 255, 256, 499]
    out = A.masked_attn(q, k, v, window=(-1, 0), prefix_lens=pre, tensor_layout="NHD")
    _compare(out, q, k, v, rows=rows, window=(-1, 0), prefix_lens=pre.tolist())
    out = A.masked_attn(q, k, v, window=(1800, 0), prefix_lens=pre, kv_lens=lens, q_offset=off, tensor_layout="NHD")
    _compare(out, q, k, v, rows=rows, window=(1800, 0), prefix_lens=pre.tolist(), kv_lens=lens.tolist(), offsets=off.tolist())
    out = A.masked_attn(q, k, v, window=(-1, 0), kv_lens=lens, q_offset="end", tensor_layout="NHD")
    _compare(out, q, k, v, rows=rows, window=(-1, 0), kv_lens=lens.tolist(), offsets=[min(n, Skv) - S for n in lens.tolist()])
    ids = torch.zeros(B, Skv, dtype=torch.int64, device=cuda)
    for cut in (1, 40, 128, 256, 300, 511, 2100, 2256, 2300):
        ids[0, cut:] += 1                                    # packed texts
    ids[1, 2200:] = -1                                       # padded tail
    ids[2] = torch.randint(-1, 3, (Skv,), device=cuda)       # any order
    ids[3] = -1                                              # nothing but padding
    for window in ((-1, -1), (-1, 0)):
        out = A.masked_attn(q, k, v, window=window, segment_ids=(ids[:, -S:], ids), tensor_layout="NHD")
        _compare(out, q, k, v, rows=[*rows, 99, 100, 199, 200], window=window, q_ids=ids[:, -S:], k_ids=ids)
        assert not out[3].any() and not out[1, 200:].any()


def test_pairs_and_hidden_garbage(cuda):
    from quantfun2_b200 import attention as A

    B, S, Skv, H, D = 4, 500, 2600, 24, 128
    q, k, v = _inputs(cuda, B, S, Skv, H, H // 2, D, BF16, seed=17)
    lens = torch.tensor([2600, 2222, 700, 0], device=cuda)
    ids = torch.zeros(B, Skv, dtype=torch.int32, device=cuda)
    ids[0, :70], ids[1, 500:], ids[2] = -1, -1, -1
    qid = torch.zeros(B, S, dtype=torch.int32, device=cuda)
    left = 1500
    j = torch.arange(Skv, device=cuda)[None]
    for kw, bad in ((dict(kv_lens=lens), j >= lens[:, None]), (dict(segment_ids=(qid, ids)), ids < 0),
                    (dict(window=(left, 0)), (j < Skv - S - left).expand(B, Skv))):
        outs = []
        for fill_k, fill_v in ((0.0, 0.0), (math.nan, math.nan), (math.inf, -math.inf)):
            kk = torch.where(bad[:, :, None, None], fill_k, k.float()).to(BF16)
            vv = torch.where(bad[:, :, None, None], fill_v, v.float()).to(BF16)
            outs.append(A.masked_attn(q, kk, vv, tensor_layout="NHD", **kw))
        assert torch.isfinite(outs[0]).all() and outs[0].any()
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, FP16)])
def test_pairs_behind_a_shared_prefix(cuda, D, dtype):
    from quantfun2_b200 import attention as A

    B, S, P, Hq, Hkv = 5, 500, 2100, 24, 8
    q, k, v, pk, pv = _inputs(cuda, B, S, S + 9, Hq, Hkv, D, dtype, seed=P, P=P)
    lens = torch.tensor([0, 1, 300, 509, 600], device=cuda)
    rows = [0, 127, 128, 256, 499]
    for kw in (dict(), dict(softcap=30.0), dict(slopes=torch.rand(Hq, device=cuda) * 0.02)):
        out = A.shared_prefix_attn(q, pk, pv, k, v, window=(-1, 0), kv_lens=lens, q_offset=9, tensor_layout="NHD", **kw)
        _compare(out, q, k, v, rows=rows, window=(-1, 0), kv_lens=lens.tolist(), offsets=[9] * B, prefix_k=pk, prefix_v=pv, **kw)


@pytest.mark.parametrize("Hq,two", [(2, False), (80, True)])
@pytest.mark.parametrize("D,dtype", [(64, FP16), (128, BF16)])
def test_scores_capped_and_biased(cuda, Hq, two, D, dtype):
    from quantfun2_b200 import attention as A

    B, S = 2, 290
    q, k, v = _inputs(cuda, B, S, S, Hq, Hq // 2, D, dtype, seed=5, amp=4.0)
    slopes = torch.rand(Hq, device=cuda) * 0.2
    rows = [0, 3, 127, 128, 200, 289]
    for R in (0, 1, 40, 700, 1024):
        table = torch.randn(Hq, 2 * R + 1, device=cuda)
        out = A.masked_attn(q, k, v, bias_table=table, tensor_layout="NHD")
        _compare(out, q, k, v, rows=rows, bias_table=table)
    for cap in (2.0, 50.0):
        out = A.masked_attn(q, k, v, window=(-1, 0), softcap=cap, tensor_layout="NHD")
        _compare(out, q, k, v, rows=rows, window=(-1, 0), softcap=cap)
        out = A.masked_attn(q, k, v, window=(50, 20), softcap=cap, slopes=slopes, sm_scale=0.3, tensor_layout="NHD")
        _compare(out, q, k, v, rows=rows, window=(50, 20), softcap=cap, slopes=slopes, sm_scale=0.3)
    out = A.masked_attn(q, k, v, slopes=slopes, tensor_layout="NHD")
    _compare(out, q, k, v, rows=rows, slopes=slopes)


@pytest.mark.parametrize("Hq,Hkv", [(2, 1), (80, 40)])
def test_bias_of_the_lowest_value_and_minus_infinity(cuda, Hq, Hkv):
    """A table of the type's lowest value everywhere weighs all keys alike; minus infinity
    hides keys; a row that has only such keys is zero."""
    from quantfun2_b200 import attention as A

    B, S, D = 2, 200, 64
    q, k, v = _inputs(cuda, B, S, S, Hq, Hkv, D, BF16, seed=8)
    low = torch.full((Hq, 3), torch.finfo(torch.float32).min, device=cuda)
    out = A.masked_attn(q, k, v, bias_table=low, tensor_layout="NHD")
    even = v.double().mean(1, keepdim=True).repeat_interleave(Hq // Hkv, 2).expand(B, S, Hq, D)
    mag = v.double().abs().mean(1, keepdim=True).repeat_interleave(Hq // Hkv, 2).expand(B, S, Hq, D)
    keys = torch.full((B, S), S, device=cuda)
    assert ((out.double() - even).abs() <= ot.attention_bound(even, mag, keys, BF16, 0.0)).all()
    past = torch.zeros(Hq, 3, device=cuda)
    past[:, 1:] = -math.inf                       # only keys strictly before the query
    out = A.masked_attn(q, k, v, bias_table=past, tensor_layout="NHD")
    _compare(out, q, k, v, rows=[1, 2, 100, 199], offsets=[-1] * B, window=(-1, 0))  # the same mask by a band
    assert not out[:, 0].any()


def test_prefix_window_and_lengths(cuda):
    from quantfun2_b200 import attention as A

    B, S, Hq, Hkv, D = 5, 270, 4, 2, 96
    q, k, v = _inputs(cuda, B, S, S, Hq, Hkv, D, BF16, seed=9)
    pre = torch.tensor([0, 1, 128, 200, 999], device=cuda)
    lens = torch.tensor([270, 0, 1, 129, 500], device=cuda, dtype=torch.int32)
    out = A.masked_attn(q, k, v, window=(-1, 0), prefix_lens=pre, tensor_layout="NHD")
    _compare(out, q, k, v, window=(-1, 0), prefix_lens=pre.tolist())
    out = A.masked_attn(q, k, v, window=(30, 0), prefix_lens=pre, kv_lens=lens, q_offset=0, tensor_layout="NHD")
    _compare(out, q, k, v, window=(30, 0), prefix_lens=pre.tolist(), kv_lens=lens.tolist(), offsets=[0] * B)
    # without a band the lengths alone matter and no offset is needed
    out = A.masked_attn(q, k, v, kv_lens=lens, tensor_layout="NHD")
    _compare(out, q, k, v, kv_lens=lens.tolist())


def test_offsets(cuda):
    from quantfun2_b200 import attention as A

    B, Sq, Skv, Hq, D = 4, 40, 300, 2, 64
    q, k, v = _inputs(cuda, B, Sq, Skv, Hq, Hq, D, BF16, seed=10)
    off = torch.tensor([-50, 0, 100, 4000], device=cuda)
    out = A.masked_attn(q, k, v, window=(60, 0), q_offset=off, tensor_layout="NHD")
    _compare(out, q, k, v, window=(60, 0), offsets=off.tolist())
    assert not out[0].any()                                  # positions before the first key
    far = torch.tensor([2 ** 31 - 1, -2 ** 31, 2 ** 30, -2 ** 30], device=cuda, dtype=torch.int32)
    out = A.masked_attn(q, k, v, window=(10, 0), q_offset=far, tensor_layout="NHD")
    assert not out.any()
    out = A.masked_attn(q, k, v, window=(-1, 0), q_offset=2 ** 40, tensor_layout="NHD")
    _compare(out, q, k, v)                                    # every key lies before such queries
    lens = torch.tensor([300, 41, 40, 3], device=cuda)
    out = A.masked_attn(q, k, v, window=(-1, 0), kv_lens=lens, q_offset="end", tensor_layout="NHD")
    _compare(out, q, k, v, window=(-1, 0), kv_lens=lens.tolist(), offsets=[n - Sq for n in lens.tolist()])


@pytest.mark.parametrize("Hq,Hkv", [(3, 1), (48, 16)])
def test_documents_and_padding(cuda, Hq, Hkv):
    from quantfun2_b200 import attention as A

    B, S, D = 4, 520, 64
    q, k, v = _inputs(cuda, B, S, S, Hq, Hkv, D, BF16, seed=11)
    ids = torch.zeros(B, S, dtype=torch.int64, device=cuda)
    for cut in (1, 40, 128, 256, 300, 511):
        ids[0, cut:] += 1                                    # packed texts
    ids[1, 200:] = -1                                        # padded tail
    ids[2] = torch.randint(-1, 3, (S,), device=cuda)         # any order
    ids[3] = -1                                              # nothing but padding
    rows = [0, 1, 39, 40, 127, 128, 199, 200, 300, 519]
    for window in ((-1, -1), (-1, 0), (64, 10)):
        out = A.masked_attn(q, k, v, window=window, segment_ids=ids, tensor_layout="NHD")
        _compare(out, q, k, v, rows=rows, window=window, q_ids=ids, k_ids=ids)
        assert not out[3].any() and not out[1, 200:].any()
    # queries and keys of unlike lengths
    out = A.masked_attn(q[:, :100], k, v, segment_ids=(ids[:, 150:250], ids), tensor_layout="NHD")
    _compare(out, q[:, :100], k, v, rows=[0, 49, 50, 99], q_ids=ids[:, 150:250], k_ids=ids)


# single tokens (and few) on caches: one to many splits, packed groups, ragged lengths
@pytest.mark.parametrize("B,Sq,Skv,Hq,Hkv,D,dtype", [
    (1, 1, 1, 4, 4, 64, BF16), (1, 1, 5000, 8, 1, 128, BF16), (3, 1, 1025, 24, 8, 96, FP16), (2, 5, 3000, 8, 4, 256, BF16),
    (16, 1, 700, 4, 2, 128, FP16), (1, 1, 40000, 2, 2, 64, BF16), (200, 1, 130, 2, 1, 64, BF16), (2, 17, 2000, 12, 1, 128, BF16),
])
def test_few_tokens_on_caches(cuda, B, Sq, Skv, Hq, Hkv, D, dtype):
    from quantfun2_b200 import attention as A

    q, k, v = _inputs(cuda, B, Sq, Skv, Hq, Hkv, D, dtype, seed=Skv)
    g = torch.Generator().manual_seed(Skv)
    lens = torch.randint(max(1, Skv // 3), Skv + 1, (B,), generator=g)
    lens[0] = Skv
    if B > 2:
        lens[1], lens[2] = 0, 1
    lens = lens.to(cuda)
    slopes = torch.rand(Hq, device=cuda) * 0.01
    table = torch.randn(Hq, 65, device=cuda)
    for kw in (dict(), dict(softcap=20.0, slopes=slopes), dict(bias_table=table)):
        out = A.masked_attn(q, k, v, window=(-1, 0), kv_lens=lens, q_offset="end", tensor_layout="NHD", **kw)
        _compare(out, q, k, v, window=(-1, 0), kv_lens=lens.tolist(), offsets=[n - Sq for n in lens.tolist()], **kw)
    out = A.masked_attn(q, k, v, window=(77, 0), kv_lens=lens, q_offset="end", tensor_layout="NHD")
    _compare(out, q, k, v, window=(77, 0), kv_lens=lens.tolist(), offsets=[n - Sq for n in lens.tolist()])


@pytest.mark.parametrize("Sq", [1, 5, 40, 100])
def test_distance_table_for_few_tokens_of_unlike_lengths(cuda, Sq):
    """One head a row, several batch elements: tile rows behind the last token belong to none."""
    from quantfun2_b200 import attention as A

    B, Skv, H, D = 3, 700, 2, 64
    q, k, v = _inputs(cuda, B, Sq, Skv, H, H, D, BF16, seed=Sq)
    lens = torch.tensor([700, 110, 333], device=cuda)
    for R in (3, 200):
        table = torch.randn(H, 2 * R + 1, device=cuda)
        out = A.masked_attn(q, k, v, window=(-1, 0), kv_lens=lens, q_offset="end", bias_table=table, tensor_layout="NHD")
        _compare(out, q, k, v, window=(-1, 0), kv_lens=lens.tolist(), offsets=[n - Sq for n in lens.tolist()],
                 bias_table=table)


def test_many_batch_elements(cuda):
    """More elements than lengths are weighed for, on caches of a few tiles."""
    from quantfun2_b200 import attention as A

    B, Skv, Hq, Hkv, D = 1500, 400, 2, 1, 64
    q, k, v = _inputs(cuda, B, 1, Skv, Hq, Hkv, D, BF16, seed=40)
    lens = torch.randint(0, Skv + 1, (B,), device=cuda, generator=torch.Generator(device=cuda).manual_seed(1))
    out = A.masked_attn(q, k, v, window=(-1, 0), kv_lens=lens, q_offset="end", tensor_layout="NHD")
    pick = [0, 1, 700, 1023, 1024, 1499]
    _compare(out[pick], q[pick], k[pick], v[pick], window=(-1, 0), kv_lens=lens[pick].tolist(),
             offsets=[n - 1 for n in lens[pick].tolist()])


def test_longest_cache_and_offsets_past_32_bits(cuda):
    """2^20 keys of 48 heads: element offsets pass 2^31, key tiles reach their limit."""
    from quantfun2_b200 import attention as A

    S, H, D = 1 << 20, 48, 64
    q = torch.randn(1, 2, H, D, device=cuda).to(BF16)
    k = torch.empty(1, S, H, D, device=cuda, dtype=BF16).normal_()
    v = torch.empty(1, S, H, D, device=cuda, dtype=BF16).normal_()
    assert k.numel() > 2 ** 31
    lens = torch.tensor([S - 77], device=cuda)
    ids = torch.zeros(1, S, dtype=torch.int32, device=cuda)
    ids[0, ::3] = 1                                            # out of order: every tile is looked at by id
    for kw, ref in ((dict(kv_lens=lens, q_offset="end", window=(-1, 0)), dict(kv_lens=[S - 77], offsets=[S - 79], window=(-1, 0))),
                    (dict(kv_lens=lens, q_offset="end", window=(300, 0)), dict(kv_lens=[S - 77], offsets=[S - 79], window=(300, 0))),
                    (dict(segment_ids=(ids[:, :2], ids)), dict(q_ids=ids[:, :2], k_ids=ids))):
        out = A.masked_attn(q, k, v, tensor_layout="NHD", **kw)
        for h in (0, H - 1):
            sl = slice(h, h + 1)
            # sums over 2^20 keys: the bound's 2^13 terms are for shorter ones; errors of fp32 sums
            # over tiles add up to 2^13 tiles * 2^-24 = 2^-11 of the sum at most, already inside it
            _compare(out[:, :, sl], q[:, :, sl], k[:, :, sl], v[:, :, sl], **ref)


@pytest.mark.parametrize("B,S,P,Hq,Hkv,D,dtype", [
    (3, 1, 1000, 4, 2, 128, BF16), (64, 1, 3001, 6, 2, 96, FP16), (5, 40, 77, 4, 4, 64, BF16), (2, 300, 130, 2, 1, 256, BF16),
    (8, 300, 260, 24, 8, 128, BF16), (130, 1, 129, 2, 2, 64, BF16), (1, 1, 1, 1, 1, 64, FP16), (9, 3, 500, 4, 1, 128, FP16),
])
def test_shared_prefix(cuda, B, S, P, Hq, Hkv, D, dtype):
    from quantfun2_b200 import attention as A

    q, k, v, pk, pv = _inputs(cuda, B, S, S + 9, Hq, Hkv, D, dtype, seed=P, P=P)
    lens = torch.randint(0, S + 10, (B,), device=cuda, generator=torch.Generator(device=cuda).manual_seed(P))
    lens[-1] = S + 9
    rows = sorted({0, S // 2, S - 1})
    slopes = torch.rand(Hq, device=cuda) * 0.02
    for kw in (dict(), dict(softcap=30.0), dict(slopes=slopes), dict(bias_table=torch.randn(Hq, 41, device=cuda))):
        out = A.shared_prefix_attn(q, pk, pv, k, v, window=(-1, 0), kv_lens=lens, q_offset=9, tensor_layout="NHD", **kw)
        _compare(out, q, k, v, rows=rows, window=(-1, 0), kv_lens=lens.tolist(), offsets=[9] * B, prefix_k=pk, prefix_v=pv,
                 **kw)
    out = A.shared_prefix_attn(q, pk, pv, k, v, window=(60, 0), tensor_layout="NHD")
    _compare(out, q, k, v, rows=rows, window=(60, 0), offsets=[9] * B, prefix_k=pk, prefix_v=pv)
    # the same keys in one cache per element
    cat_k = torch.cat([pk.expand(B, P, Hkv, D), k], 1)
    cat_v = torch.cat([pv.expand(B, P, Hkv, D), v], 1)
    hnd = A.shared_prefix_attn(q.transpose(1, 2), pk.transpose(0, 1), pv.transpose(0, 1), k.transpose(1, 2),
                               v.transpose(1, 2), window=(-1, 0))
    _compare(hnd.transpose(1, 2), q, cat_k, cat_v, rows=rows, window=(-1, 0))


def test_no_keys_and_no_queries(cuda):
    from quantfun2_b200 import attention as A

    for Sq in (1, 300):
        q, k, v = _inputs(cuda, 2, Sq, 0, 80, 80, 64, BF16)
        out = torch.full_like(q, 7.0)
        assert A.masked_attn(q, k, v, window=(-1, 0), tensor_layout="NHD", out=out) is out and not out.any()
        ids = (torch.zeros(2, Sq, device=cuda, dtype=torch.int32), torch.zeros(2, 0, device=cuda, dtype=torch.int32))
        out = A.masked_attn(q, k, v, segment_ids=ids, tensor_layout="NHD")
        assert out.shape == q.shape and not out.any()
    q, k, v, pk, pv = _inputs(cuda, 2, 5, 0, 2, 2, 64, BF16, P=30)
    out = A.shared_prefix_attn(q, pk, pv, k, v, tensor_layout="NHD")
    _compare(out, q, k, v, rows=[0, 4], offsets=[0, 0], prefix_k=pk, prefix_v=pv)
    out = A.shared_prefix_attn(q, pk[:0], pv[:0], k, v, tensor_layout="NHD")
    assert not out.any()
    assert A.masked_attn(q[:, :0], k, v, tensor_layout="NHD").shape == (2, 0, 2, 64)
    assert A.masked_attn(q[:0], k[:0], v[:0], tensor_layout="NHD").shape == (0, 5, 2, 64)


@pytest.mark.parametrize("Sq,Hq", [(1, 4), (200, 4), (300, 80)])
def test_hidden_garbage_changes_nothing(cuda, Sq, Hq):
    """Infinities and NaN in keys that no row sees: behind the lengths, in padding, before the
    window; the bits of the result are those with zeros there."""
    from quantfun2_b200 import attention as A

    B, Skv, D = 2, 700, 128
    q, k, v = _inputs(cuda, B, Sq, Skv, Hq, Hq // 2, D, BF16, seed=13)
    lens = torch.tensor([650, 333], device=cuda)
    ids = torch.zeros(B, Skv, dtype=torch.int32, device=cuda)
    ids[0, :70], ids[1, 500:] = -1, -1
    qid = torch.zeros(B, Sq, dtype=torch.int32, device=cuda)
    left = 100
    first = [n - Sq - left for n in lens.tolist()]
    calls = [
        (dict(kv_lens=lens), lambda b, j: j >= lens[b]),
        (dict(segment_ids=(qid, ids)), lambda b, j: ids[b] < 0),
        (dict(kv_lens=lens, q_offset="end", window=(left, 0)), lambda b, j: (j >= lens[b]) | (j < first[b])),
    ]
    j = torch.arange(Skv, device=cuda)
    for kw, hidden in calls:
        bad = torch.stack([hidden(b, j) for b in range(B)])
        assert bad.any()
        outs = []
        for fill_k, fill_v in ((0.0, 0.0), (math.nan, math.nan), (math.inf, -math.inf)):
            kk = torch.where(bad[:, :, None, None], fill_k, k.float()).to(BF16)
            vv = torch.where(bad[:, :, None, None], fill_v, v.float()).to(BF16)
            outs.append(A.masked_attn(q, kk, vv, tensor_layout="NHD", **kw))
        assert torch.isfinite(outs[0]).all() and outs[0].any()
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_seen_nan_reaches_its_rows(cuda):
    from quantfun2_b200 import attention as A

    q, k, v = _inputs(cuda, 1, 1, 3000, 2, 2, 64, BF16, seed=14)
    k[0, 2100, 1, 3] = math.nan
    out = A.masked_attn(q, k, v, tensor_layout="NHD")
    assert out[0, 0, 1].isnan().all() and torch.isfinite(out[0, 0, 0]).all()


def test_strided_inputs_and_outputs(cuda):
    from quantfun2_b200 import attention as A

    B, S, H, D = 2, 150, 3, 64
    joint = torch.randn(B, S, 3 * H, D + 8, device=cuda).to(BF16)
    q, k, v = (joint[:, :, n * H:(n + 1) * H, :D] for n in range(3))
    buf = torch.full((B, S + 5, 2 * H, D), 3.0, device=cuda, dtype=BF16)
    out = buf[:, 2:S + 2, H:]
    assert A.masked_attn(q, k, v, window=(-1, 0), tensor_layout="NHD", out=out) is out
    _compare(out, q, k, v, rows=[0, 64, 149], window=(-1, 0))
    rest = buf.clone()
    rest[:, 2:S + 2, H:] = 3.0
    assert (rest == 3.0).all()                             # nothing beside the view was written
    odd = torch.randn(B, S, 3 * H, D + 1, device=cuda).to(BF16)[..., 1:]     # rows off the 16-byte alignment
    out = A.masked_attn(odd[:, :, :H], odd[:, :, H:2 * H], odd[:, :, 2 * H:], tensor_layout="NHD")
    _compare(out, odd[:, :, :H], odd[:, :, H:2 * H], odd[:, :, 2 * H:], rows=[0, 149])
    one = k[:1].expand(B, S, H, D)                         # one batch element's keys for all
    out = A.masked_attn(q, one, v[:1].expand(B, S, H, D), tensor_layout="NHD")
    _compare(out, q, one, v[:1].expand(B, S, H, D), rows=[0, 149])


def test_two_streams_and_a_graph(cuda):
    """Calls at once on two streams, and a captured call replayed on other lengths and values:
    the bits of the calls alone."""
    from quantfun2_b200 import attention as A

    sets = [_inputs(cuda, 2, 1, 9000, 8, 2, 128, BF16, seed=20 + n) for n in range(2)]
    lens = [torch.tensor([9000, 4000], device=cuda, dtype=torch.int32), torch.tensor([77, 8999], device=cuda, dtype=torch.int32)]
    call = lambda n: A.masked_attn(*sets[n], window=(-1, 0), kv_lens=lens[n], q_offset="end", tensor_layout="NHD")  # noqa: E731
    alone = [call(n) for n in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[n].append(call(n))
    torch.cuda.synchronize()
    for n in range(2):
        assert all(torch.equal(o, alone[n]) for o in got[n])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = call(0)
    for t, u in zip(sets[0], sets[1]):
        t.copy_(u)
    lens[0].copy_(lens[1])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, alone[1])
    A.masked_attn_status()


def test_prompt_then_tokens_then_shared_prefix(cuda):
    """A run as an encoder-decoder of texts would make it: rotate, store, attend for a prompt;
    then token by token on the cache; then the prompt as the shared prefix of three answers."""
    from quantfun2_b200 import attention as A
    from quantfun2_b200 import kernels as K

    Hq, Hkv, D, S, more = 6, 2, 128, 150, 4
    g = torch.Generator(device=cuda).manual_seed(30)
    f = K.rotary_inv_freq(64, device=cuda)
    tok = lambda n, B=1: [torch.randn(B, n, h, D, device=cuda, generator=g).to(BF16) for h in (Hq, Hkv, Hkv)]  # noqa: E731
    cache_k = torch.full((1, 256, Hkv, D), math.nan, device=cuda, dtype=BF16)   # the unused end holds garbage
    cache_v = torch.full_like(cache_k, math.nan)
    kw = dict(window=(-1, 0), softcap=30.0, tensor_layout="NHD")
    q, k, v = tok(S)
    q, k = K.rotary_apply(q, k, torch.arange(S, device=cuda), f)
    cache_k[:, :S], cache_v[:, :S] = k, v
    out = A.masked_attn(q, k, v, **kw)
    _compare(out, q, k, v, rows=[0, 128, S - 1], window=(-1, 0), softcap=30.0)
    lens = torch.tensor([S], device=cuda, dtype=torch.int32)
    for n in range(more):
        q, k, v = tok(1)
        K.rotary_apply_(q, k, torch.full((1, 1), S + n, device=cuda), f)
        cache_k[:, S + n], cache_v[:, S + n] = k[:, 0], v[:, 0]
        lens += 1
        out = A.masked_attn(q, cache_k, cache_v, kv_lens=lens, q_offset="end", **kw)
        _compare(out, q, cache_k[:, :S + n + 1], cache_v[:, :S + n + 1], window=(-1, 0), softcap=30.0)
    B, P = 3, S + more
    q, k, v = tok(7, B)
    pos = P + torch.arange(7, device=cuda)
    q, k = K.rotary_apply(q, k, pos, f)
    own = torch.tensor([7, 5, 6], device=cuda)
    out = A.shared_prefix_attn(q, cache_k[0, :P], cache_v[0, :P], k, v, kv_lens=own, q_offset=0, **kw)
    _compare(out, q, k, v, window=(-1, 0), softcap=30.0, kv_lens=own.tolist(), offsets=[0] * B, prefix_k=cache_k[0, :P],
             prefix_v=cache_v[0, :P])


def test_do_attn_masked_backend(cuda):
    from quantfun2_b200 import attention as A

    B, S, Hq, Hkv, D = 3, 300, 6, 2, 96
    q, k, v = _inputs(cuda, B, S, S, Hq, Hkv, D, BF16, seed=31)
    mask = torch.ones(B, S, dtype=torch.bool, device=cuda)
    mask[1, 200:] = False
    mask[2] = torch.rand(S, device=cuda) < 0.5
    A.ATTN = "masked"
    try:
        out = A.do_attn(None, q, k, v, mask)
        dense = A.do_attn(None, q, k, v, None)
    finally:
        A.ATTN = "b200"
    ids = mask.int() - 1
    _compare(out, q, k, v, rows=[0, 100, 199, 200, 299], q_ids=ids, k_ids=ids)
    assert not out[~mask].any()
    _compare(dense, q, k, v, rows=[0, 299])


def test_refusals(cuda):
    from quantfun2_b200 import attention as A

    q, k, v = _inputs(cuda, 2, 4, 8, 4, 2, 64, BF16)
    nhd = dict(tensor_layout="NHD")
    i32 = lambda *x: torch.tensor(x, device=cuda, dtype=torch.int32)  # noqa: E731
    with pytest.raises(A.QF2Error):
        A.masked_attn(q.float(), k.float(), v.float(), **nhd)
    bad = [
        ((q, k.half(), v), {}), ((q, k, v[:, :7]), {}), ((q, k[:1], v[:1]), {}), ((q[0], k, v), {}),
        ((q[..., :56], k[..., :56], v[..., :56]), {}), ((q[:, :, :3], k, v), {}), ((q.cpu(), k, v), {}),
        ((q, k, v), dict(tensor_layout="other")), ((q, k, v), dict(kv_lens=i32(1))), ((q, k, v), dict(kv_lens=i32(1, 1).cpu())),
        ((q, k, v), dict(kv_lens=i32(1, 1).float())), ((q, k, v), dict(kv_lens=i32(1, 1), window=(-1, 0))),
        ((q, k, v), dict(q_offset="start")), ((q, k, v), dict(q_offset=i32(1))), ((q, k, v), dict(segment_ids=torch.zeros(2, 4, device=cuda, dtype=torch.int32))),
        ((q, k, v), dict(softcap=-1.0)), ((q, k, v), dict(softcap=math.inf)), ((q, k, v), dict(sm_scale=0.0)),
        ((q, k, v), dict(slopes=torch.ones(2, device=cuda))), ((q, k, v), dict(slopes=torch.ones(4, device=cuda).half())),
        ((q, k, v), dict(bias_table=torch.ones(4, 4, device=cuda))), ((q, k, v), dict(bias_table=torch.ones(4, 2051, device=cuda))),
        ((q, k, v), dict(slopes=torch.ones(4, device=cuda), bias_table=torch.ones(4, 3, device=cuda))),
        ((q, k, v), dict(out=torch.empty(2, 4, 4, 64, device=cuda))), ((q, k, v), dict(out=torch.empty(2, 5, 4, 64, device=cuda, dtype=BF16))),
        ((q, k, v), dict(out=torch.empty(2, 4, 4, 68, device=cuda, dtype=BF16)[..., :64])),
        ((q.requires_grad_(), k, v), {}),
    ]
    for args, kw in bad:
        with pytest.raises(A.QF2Error):
            A.masked_attn(*args, **{**nhd, **kw})
    q = q.detach()
    pk = k[0]
    for args in ((q, None, None, k, v), (q, pk, None, k, v), (q, pk[None], pk[None], k, v), (q, pk[:, :1], pk[:, :1], k, v),
                 (q, pk[..., :32], pk[..., :32], k, v), (q, pk.half(), pk.half(), k, v)):
        with pytest.raises(A.QF2Error):
            A.shared_prefix_attn(*args, **nhd)
    with torch.no_grad():                                    # a parameter's values are fine where no gradient is wanted
        A.masked_attn(q.clone().requires_grad_(), k, v, **nhd)
    A.masked_attn_status()


@pytest.mark.parametrize("B,Sq,Skv,Hq,Hkv,D,dtype", [
    (2, 1, 1500, 24, 8, 64, BF16), (3, 5, 700, 6, 2, 128, FP16), (2, 6, 700, 6, 2, 128, BF16), (1, 300, 300, 6, 2, 96, BF16),
    (2, 100, 900, 16, 1, 256, BF16), (4, 1, 2000, 40, 1, 128, FP16),
])
def test_distance_table_of_grouped_heads(cuda, B, Sq, Skv, Hq, Hkv, D, dtype):
    """Tables within and beyond their reach, their last entries minus infinity or unlike each
    other, for heads that share keys."""
    from quantfun2_b200 import attention as A

    q, k, v = _inputs(cuda, B, Sq, Skv, Hq, Hkv, D, dtype, seed=Sq + Skv)
    rows = sorted({0, Sq // 2, Sq - 1})
    g = torch.Generator(device=cuda).manual_seed(3)
    for R in (0, 3, 150, 1024):
        table = torch.randn(Hq, 2 * R + 1, device=cuda, generator=g)
        table[:, 0] += 2.0
        table[:, -1] -= 2.0
        for window in ((-1, 0), (-1, -1)):
            out = A.masked_attn(q, k, v, window=window, bias_table=table, tensor_layout="NHD")
            _compare(out, q, k, v, rows=rows, window=window, bias_table=table)
    table = torch.randn(Hq, 9, device=cuda, generator=g)
    table[:, 0] = -math.inf                                  # keys 4 and more before the query are hidden
    out = A.masked_attn(q, k, v, window=(-1, 0), bias_table=table, tensor_layout="NHD")
    _compare(out, q, k, v, rows=rows, window=(3, 0), bias_table=torch.where(table.isinf(), 0.0, table))


@pytest.mark.parametrize("D,dtype", [(64, BF16), (96, FP16), (128, BF16), (256, FP16)])
def test_many_rows_of_split_keys(cuda, D, dtype):
    """More rows than are merged by a block each; elements without keys, splits without keys."""
    from quantfun2_b200 import attention as A

    B, Sq, Skv, H = 2, 128, 6000, 12
    q, k, v = _inputs(cuda, B, Sq, Skv, H, H, D, dtype, seed=D)
    for lens in ([6000, 6000], [6000, 0], [200, 5000]):
        lens = torch.tensor(lens, device=cuda)
        out = A.masked_attn(q, k, v, window=(-1, 0), kv_lens=lens, q_offset="end", tensor_layout="NHD")
        _compare(out, q, k, v, rows=[0, 1, 64, 127], window=(-1, 0), kv_lens=lens.tolist(),
                 offsets=[n - Sq for n in lens.tolist()])
    out = A.masked_attn(q, k, v, tensor_layout="NHD")
    _compare(out, q, k, v, rows=[0, 127])
    assert torch.equal(out, A.masked_attn(q, k, v, tensor_layout="NHD"))


@pytest.mark.parametrize("B,Sq,Hq,Hkv,D,dtype", [(64, 1, 24, 8, 128, BF16), (2, 16, 8, 4, 256, FP16), (1, 300, 12, 12, 64, BF16)])
def test_narrow_windows_on_long_caches(cuda, B, Sq, Hq, Hkv, D, dtype):
    from quantfun2_b200 import attention as A

    Skv = 5000
    q, k, v = _inputs(cuda, B, Sq, Skv, Hq, Hkv, D, dtype, seed=50)
    lens = torch.randint(Sq, Skv + 1, (B,), device=cuda, generator=torch.Generator(device=cuda).manual_seed(2))
    pick, rows = sorted({0, B // 2, B - 1}), sorted({0, Sq // 2, Sq - 1})
    for window in ((0, 0), (127, 0), (700, 0), (90, 40)):
        out = A.masked_attn(q, k, v, window=window, kv_lens=lens, q_offset="end", tensor_layout="NHD")
        _compare(out[pick], q[pick], k[pick], v[pick], rows=rows, window=window, kv_lens=lens[pick].tolist(),
                 offsets=[n - Sq for n in lens[pick].tolist()])
        out = A.masked_attn(q, k, v, window=window, tensor_layout="NHD")
        _compare(out[pick], q[pick], k[pick], v[pick], rows=rows, window=window)


def test_lengths_and_offsets_in_64_bits(cuda):
    """Beyond 32 bits: all keys, the far end; below zero: none."""
    from quantfun2_b200 import attention as A

    B, Sq, Skv = 5, 9, 300
    q, k, v = _inputs(cuda, B, Sq, Skv, 2, 1, 64, BF16, seed=60)
    lens = torch.tensor([2 ** 32 + 3, 2 ** 31, -2 ** 33, 2 ** 40, 5], device=cuda)
    _compare(A.masked_attn(q, k, v, kv_lens=lens, tensor_layout="NHD"), q, k, v, kv_lens=lens.tolist())
    off = torch.tensor([2 ** 40, -2 ** 40, 2 ** 32, 2 ** 32 - 1, 100], device=cuda)
    out = A.masked_attn(q, k, v, window=(50, 0), q_offset=off, tensor_layout="NHD")
    _compare(out, q, k, v, window=(50, 0), offsets=off.tolist())
    out = A.masked_attn(q, k, v, window=(-1, 0), q_offset=off, prefix_lens=lens, tensor_layout="NHD")
    _compare(out, q, k, v, window=(-1, 0), offsets=off.tolist(), prefix_lens=lens.tolist())


@pytest.mark.parametrize("B,Sq,Skv,Hq,Hkv,D,dtype", [
    (3, 5, 300, 4, 2, 64, BF16), (3, 200, 500, 6, 2, 96, FP16), (3, 400, 900, 40, 8, 64, BF16), (4, 500, 2500, 24, 8, 128, FP16),
    (3, 40, 300, 2, 1, 256, BF16)])
def test_ids_in_64_bits(cuda, B, Sq, Skv, Hq, Hkv, D, dtype):
    """Ids that share their low or their high words are unlike, in order and out of order; beside
    int32 ones, and where only the queries' are wide."""
    from quantfun2_b200 import attention as A

    q, k, v = _inputs(cuda, B, Sq, Skv, Hq, Hkv, D, dtype, seed=61)
    names = torch.tensor([5, 2 ** 31, 2 ** 32 + 5, 2 ** 33 + 5, 2 ** 33 + 6, 2 ** 63 - 1, -1, -2 ** 63], device=cuda)
    g = torch.Generator(device=cuda).manual_seed(62)
    pick = lambda n, of: torch.randint(0, of, (B, n), device=cuda, generator=g)  # noqa: E731
    rows = sorted({0, 1, Sq // 3, Sq // 2, Sq - 2, Sq - 1})
    ki, qi = names[pick(Skv, 8).sort(1).values], names[pick(Sq, 8)]
    mixed = names[pick(Skv, 8)]
    mixed[1] = torch.where(mixed[1] > 2 ** 31 - 1, 7, mixed[1])          # an element of narrow ids
    narrow = torch.randint(-1, 6, (B, Skv), device=cuda, generator=g)
    for qq, kk in ((qi, ki), (qi, mixed), (qi, narrow), (qi, narrow.int()), (narrow[:, :Sq].int(), mixed), (narrow[:, :Sq], narrow)):
        for window in ((-1, -1), (150, 30)):
            out = A.masked_attn(q, k, v, window=window, segment_ids=(qq, kk), tensor_layout="NHD")
            _compare(out, q, k, v, rows=rows, window=window, q_ids=qq.long(), k_ids=kk.long())
    a = A.masked_attn(q, k, v, segment_ids=(narrow[:, :Sq], narrow), tensor_layout="NHD")
    b = A.masked_attn(q, k, v, segment_ids=(narrow[:, :Sq].int(), narrow.int()), tensor_layout="NHD")
    assert torch.equal(a, b)


@pytest.mark.parametrize("Sq,Skv,Hq,D,dtype", [(1, 700, 4, 128, BF16), (5, 700, 4, 64, FP16), (200, 700, 4, 128, BF16), (300, 700, 80, 64, BF16),
                                               (150, 700, 4, 256, FP16), (500, 2600, 48, 96, BF16)])
def test_hidden_keys_choose_no_arithmetic_of_capped_scores(cuda, Sq, Skv, Hq, D, dtype):
    """Great finite values behind the lengths, in padding and outside the window change no bit of
    capped scores; neither does what an earlier kernel left in shared memory."""
    from quantfun2_b200 import attention as A

    B = 2
    q, k, v = _inputs(cuda, B, Sq, Skv, Hq, Hq // 2, D, dtype, seed=63)
    lens = torch.tensor([Skv - 50, Skv // 2], device=cuda)
    ids = torch.zeros(B, Skv, dtype=torch.int32, device=cuda)
    ids[0, :70], ids[1, Skv // 2:] = -1, -1
    qid = torch.zeros(B, Sq, dtype=torch.int32, device=cuda)
    j = torch.arange(Skv, device=cuda)[None]
    left = 300
    calls = [(dict(kv_lens=lens), j >= lens[:, None]), (dict(segment_ids=(qid, ids)), ids < 0),
             (dict(window=(left, 0)), (j < Skv - Sq - left).expand(B, Skv))]
    for kw, hidden in calls:
        outs = []
        for fill in (0.0, 1e3, -1e3, math.nan):
            kk = torch.where(hidden[:, :, None, None], fill, k.float()).to(dtype)
            A.masked_attn(q * 30, k * 30, v, tensor_layout="NHD")        # large values in every block's memory
            outs.append(A.masked_attn(q, kk, v, softcap=50.0, tensor_layout="NHD", **kw))
        assert outs[0].any()
        assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("cap", [0.5, 50.0, 1e3, 1e6, 1e15, 1e30, 1e38])
@pytest.mark.parametrize("Sq,Hq,D,dtype", [(2, 2, 64, BF16), (130, 4, 128, FP16), (300, 80, 64, BF16), (70, 4, 256, BF16)])
def test_caps_of_every_size(cuda, cap, Sq, Hq, D, dtype):
    """A cap far above the scores leaves them as they are, in tiles with rows that do not exist
    and beside a row whose scores reach the cap."""
    from quantfun2_b200 import attention as A

    q, k, v = _inputs(cuda, 1, Sq, 192, Hq, Hq // 2, D, dtype, seed=64)
    q[:, 0] *= 200
    rows = sorted({1, Sq // 2, Sq - 1})
    _compare(A.masked_attn(q, k, v, softcap=cap, tensor_layout="NHD"), q, k, v, rows=rows, softcap=cap)


@pytest.mark.parametrize("Sq,Hq,Hkv,D,dtype", [(2, 2, 1, 64, BF16), (2, 40, 20, 128, FP16), (200, 4, 2, 96, BF16), (200, 4, 2, 256, FP16), (300, 80, 40, 64, FP16),
                                               (600, 40, 40, 128, BF16)])
@pytest.mark.parametrize("wide", [False, True])
def test_keys_of_ids_without_queries_hold_garbage(cuda, Sq, Hq, Hkv, D, dtype, wide):
    """Keys of an id between two ids of a tile's queries, that no query has, do not enter: the bits
    of the result are those with zeros there.  In order and out of order; 64-bit ids with equal low words."""
    from quantfun2_b200 import attention as A

    B, Skv = 3, 700
    q, k, v = _inputs(cuda, B, Sq, Skv, Hq, Hkv, D, dtype, seed=70)
    g = torch.Generator(device=cuda).manual_seed(71)
    ki = torch.arange(Skv, device=cuda)[None].expand(B, Skv) * 7 // Skv              # 0 .. 6, in order
    qi = torch.randint(0, 4, (B, Sq), device=cuda, generator=g) * 2                  # even ones
    if Sq > 2:
        qi[1, 50:] = -1                                                              # few queries, others padding
    qi[0] = qi[0].sort().values
    perm = torch.randperm(Skv, device=cuda, generator=g)
    name = (lambda x: torch.where(x < 0, x, 5 + x * 2 ** 32)) if wide else (lambda x: x.int())
    for kid in (ki, ki[:, perm]):
        hidden = torch.stack([~torch.isin(kid[b], qi[b]) for b in range(B)])
        assert hidden.any(1).all()
        outs = []
        for fill in (0.0, math.nan, math.inf, -math.inf):
            vv = torch.where(hidden[:, :, None, None], fill, v.float()).to(dtype)
            outs.append(A.masked_attn(q, k, vv, segment_ids=(name(qi), name(kid)), tensor_layout="NHD"))
        assert torch.isfinite(outs[0]).all() and outs[0].any()
        assert all(torch.equal(outs[0], o) for o in outs[1:])
        rows = sorted({0, Sq // 2, Sq - 1})
        vv = torch.where(hidden[:, :, None, None], 0.0, v.float()).to(dtype)
        _compare(outs[0], q, k, vv, rows=rows, q_ids=qi, k_ids=kid)


def test_keys_between_bands_hold_garbage(cuda):
    """Queries with padding between them and narrow windows; batch elements at far positions of one
    shared prefix: what lies between their bands does not enter."""
    from quantfun2_b200 import attention as A

    for Hq, D in ((2, 64), (24, 128)):
        S = 300
        q, k, v = _inputs(cuda, 2, S, S, Hq, Hq, D, BF16, seed=72)
        qi = torch.full((2, S), -1, device=cuda, dtype=torch.int32)
        qi[0, [5, 6, 100, 290]] = 0
        qi[1, [0, 299]] = 3
        for ki in (torch.tensor([0, 3], device=cuda, dtype=torch.int32)[:, None].expand(2, S),
                   torch.where(torch.arange(S, device=cuda) % 50 == 0, -1, torch.tensor([0, 3], device=cuda)[:, None]).int()):
            t = torch.arange(S, device=cuda)
            band = (t[:, None] - t[None]).abs() <= 2                       # [queries, keys]
            hidden = torch.stack([~(band & (qi[b, :, None] == ki[b][None]) & (qi[b, :, None] >= 0)).any(0) for b in range(2)])
            outs = [A.masked_attn(q, k, torch.where(hidden[:, :, None, None], f, v.float()).to(BF16), window=(2, 2),
                                  segment_ids=(qi, ki), tensor_layout="NHD") for f in (0.0, math.nan, math.inf)]
            assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2]) and outs[0].any()
        B, P = 6, 900
        q, k, v, pk, pv = _inputs(cuda, B, 1, 4, Hq, Hq, D, BF16, seed=73, P=P)
        at = torch.tensor([10, 890, 130, 500, 10, 2], device=cuda)         # positions in the prefix
        for dist in (3, 60):
            j = torch.arange(P, device=cuda)
            hidden = ~((j[None] <= at[:, None]) & (j[None] >= at[:, None] - dist)).any(0)
            outs = [A.shared_prefix_attn(q, pk, torch.where(hidden[:, None, None], f, pv.float()).to(BF16), k, v, window=(dist, 0),
                                         q_offset=at - P, tensor_layout="NHD") for f in (0.0, math.nan, -math.inf)]
            assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2]) and outs[0].any()


@pytest.mark.parametrize("Sq,Skv,Hq,Hkv,D,dtype", [(1, 3000, 4, 2, 64, BF16), (5, 300, 4, 2, 128, FP16), (140, 500, 4, 4, 96, BF16), (300, 700, 80, 80, 64, BF16),
                                                    (500, 2600, 48, 48, 128, FP16)])
def test_slopes_of_far_queries(cuda, Sq, Skv, Hq, Hkv, D, dtype):
    """Queries millions of positions from their keys, on both sides: the weights follow from the
    keys' distances to each other."""
    from quantfun2_b200 import attention as A

    B = 3
    q, k, v = _inputs(cuda, B, Sq, Skv, Hq, Hkv, D, dtype, seed=74)
    slopes = torch.rand(Hq, device=cuda) * 0.5 + 0.01
    rows = sorted({0, Sq // 2, Sq - 1})
    for off in ([2 ** 22, 2 ** 28 + 3, 10 ** 6], [-2 ** 28, -10 ** 6 - 1, -2 ** 22], [Skv, -Sq, 0]):
        at = torch.tensor(off, device=cuda)
        lens = torch.tensor([Skv, Skv // 2, Skv - 1], device=cuda)
        for kw in (dict(), dict(kv_lens=lens), dict(prefix_lens=torch.tensor([7, 200, 0], device=cuda), window=(50, 50))):
            out = A.masked_attn(q, k, v, slopes=slopes, q_offset=at, tensor_layout="NHD", **kw)
            _compare(out, q, k, v, rows=rows, slopes=slopes, offsets=off, **{n: x.tolist() if hasattr(x, "tolist") else x for n, x in kw.items()})
    P = 700
    pk, pv = torch.randn(P, Hkv, D, device=cuda).to(dtype), torch.randn(P, Hkv, D, device=cuda).to(dtype)
    out = A.shared_prefix_attn(q, pk, pv, k, v, slopes=slopes, q_offset=2 ** 27, tensor_layout="NHD")
    _compare(out, q, k, v, rows=rows, slopes=slopes, offsets=[2 ** 27] * B, prefix_k=pk, prefix_v=pv)


@pytest.mark.parametrize("cap", [5e-324, 1e-42, 1e-38, 1e-20])
def test_caps_near_zero(cuda, cap):
    """All scores but zeros are at the cap, which is nothing: an even softmax, with zero rows of q too."""
    from quantfun2_b200 import attention as A

    for Sq, Hq in ((2, 2), (300, 80)):
        q, k, v = _inputs(cuda, 1, Sq, 200, Hq, Hq, 64, BF16, seed=75)
        q[:, 0] = 0.0
        _compare(A.masked_attn(q, k, v, softcap=cap, tensor_layout="NHD"), q, k, v, rows=[0, Sq - 1], softcap=cap)


@pytest.mark.parametrize("B,S,H,D,dtype", [(2, 1, 4, 64, BF16), (1, 40, 4, 128, FP16), (3, 300, 40, 64, BF16), (2, 2500, 24, 128, BF16), (2, 300, 4, 256, BF16)])
def test_out_over_the_inputs(cuda, B, S, H, D, dtype):
    """Into q, k or v themselves, into parts of them, and beside them in one buffer."""
    from quantfun2_b200 import attention as A

    q, k, v = _inputs(cuda, B, S, S, H, H, D, dtype, seed=76)
    kw = dict(window=(-1, 0), tensor_layout="NHD")
    want = A.masked_attn(q, k, v, **kw)
    for n in range(3):
        t = [x.clone() for x in (q, k, v)]
        assert A.masked_attn(*t, out=t[n], **kw) is t[n] and torch.equal(t[n], want)
    joint = torch.cat([q, k, v, v], 2)
    for n in range(4):                                                # q's, k's, v's and the last heads
        j = joint.clone()
        qq, kk, vv, rest = j.split(H, 2)
        out = (qq, kk, vv, rest)[n]
        assert A.masked_attn(qq, kk, vv, out=out, **kw) is out and torch.equal(out, want)
        keep = [m for m in range(4) if m != n]
        assert all(torch.equal(j.split(H, 2)[m], joint.split(H, 2)[m]) for m in keep)
    j = joint.clone()
    qq, kk, vv, _ = j.split(H, 2)
    out = j[:, :, H // 2:H // 2 + H]                                  # half over q, half over k
    assert torch.equal(A.masked_attn(qq, kk, vv, out=out, **kw), want)
    P = 200
    pk, pv = torch.randn(B * S + P, H, D, device=cuda).to(dtype), torch.randn(P, H, D, device=cuda).to(dtype)
    want = A.shared_prefix_attn(q, pk[:P], pv, k, v, **kw)
    out = pk[:B * S].view(B, S, H, D)                                 # over the prefix's keys
    assert torch.equal(A.shared_prefix_attn(q, pk[:P], pv, k, v, out=out, **kw), want)
    with pytest.raises(A.QF2Error):
        A.masked_attn(q, k, v, out=torch.empty(B * S * H * D, device=cuda, dtype=dtype).as_strided(q.shape, (0 if B > 1 else H * D, H * D, D // 2, 1)), **kw)


def test_do_attn_masked_takes_masks_of_any_type(cuda):
    """What is not zero is a token, as for the other backends."""
    from quantfun2_b200 import attention as A

    q, k, v = _inputs(cuda, 2, 90, 90, 4, 2, 64, BF16, seed=77)
    mask = torch.rand(2, 90, device=cuda) < 0.7
    A.ATTN = "masked"
    try:
        want = A.do_attn(None, q, k, v, mask)
        for m in (mask.int(), mask.float() * 0.5, mask.to(torch.uint8) * torch.arange(1, 91, device=cuda, dtype=torch.uint8), -mask.long()):
            assert torch.equal(A.do_attn(None, q, k, v, m), want)
    finally:
        A.ATTN = "b200"
