"""GPU: which keys masked attention and its shared-prefix form count, each exactly once.

Queries are zero, so all seen keys weigh the same: the weights are 1, the sums are whole numbers
below 2^24 that fp32 holds exactly, and the result is sum_seen v / n with one division (two fp32
roundings of 2^-24) and one rounding to the type.  A key that is left out, counted twice or seen
by mistake changes it by far more where V has little else: single keys at the edges of masks,
tiles and splits, each alone in a channel, or tiles whose values add up to +-128 a channel."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def _seen(dev, B, Sq, Skv, P=0, window=(-1, -1), offsets=None, kv_lens=None, prefix_lens=None, q_ids=None, k_ids=None):
    """[B, Sq, P + Skv] truth values from the definition."""
    j = torch.arange(P + Skv, device=dev)[None, None]
    off = torch.tensor([Skv - Sq] * B if offsets is None else offsets, device=dev)
    t = (P + off[:, None] + torch.arange(Sq, device=dev)[None])[:, :, None]
    band = torch.ones(B, Sq, P + Skv, dtype=torch.bool, device=dev)
    if window[0] >= 0:
        band &= j >= t - window[0]
    if window[1] >= 0:
        band &= j <= t + window[1]
    if prefix_lens is not None:
        band |= j < torch.tensor(prefix_lens, device=dev)[:, None, None]
    if kv_lens is not None:
        band &= j < P + torch.tensor(kv_lens, device=dev).clamp(0, Skv)[:, None, None]
    if q_ids is not None:
        band &= (q_ids[:, :, None] == k_ids[:, None]) & (q_ids >= 0)[:, :, None]
    return band


def _edges(seen, D):
    """Keys around the edges of the first, middle and last rows' masks, of tiles and of the store;
    at most D, those of the masks first."""
    B, Sq, n = seen.shape
    first = []
    for b in sorted({0, B // 2, B - 1}):
        for i in sorted({0, Sq // 2, Sq - 1}):
            row = seen[b, i].int()
            turn = (row[1:] != row[:-1]).nonzero().flatten().tolist()
            for x in turn[:3] + turn[-3:]:
                first += [x, x + 1]
    tiles = (n + 127) // 128
    for t in sorted({0, 1, tiles // 3, tiles // 2, tiles - 2, tiles - 1}):
        first += [128 * t - 1, 128 * t, 128 * t + 63, 128 * t + 64, 128 * t + 95, 128 * t + 96, 128 * t + 31, 128 * t + 32]
    first += [0, n - 1, n - 2] + list(range(n - 1, -1, -max(1, n // D)))
    keys = []
    for x in first:
        if 0 <= x < n and x not in keys:
            keys.append(x)
    return keys[:D]


def _check(call, seen, Hkv, D, dtype, P=0):
    """call(k, v, prefix_k, prefix_v) -> out [B, Sq, Hq, D] for zero queries."""
    from quantfun2_b200 import attention as A

    dev = seen.device
    B, Sq, n = seen.shape
    g = torch.Generator(device=dev).manual_seed(n)
    lone = torch.zeros(n, D, device=dev)
    for c, x in enumerate(_edges(seen, D)):
        lone[x, c] = 2.0 ** min(15, max(0, n.bit_length() - 1))
    signs = torch.randint(0, 2, (n // 128 + 1, D), device=dev, generator=g).float() * 2 - 1
    tiles = signs.repeat_interleave(128, 0)[:n]
    count = seen.sum(-1, keepdim=True).double()
    for vals in (lone, tiles):
        # the same for all heads, turned by one channel a head, so that heads cannot be mistaken
        v = torch.stack([vals.roll(h, -1) for h in range(Hkv)], 1).to(dtype)                   # [n, Hkv, D]
        k = torch.randn(n, Hkv, D, device=dev, generator=g).to(dtype)
        own = lambda t: t[None, P:].expand(B, n - P, Hkv, D).contiguous()  # noqa: E731
        out = call(own(k), own(v), k[:P], v[:P])
        A.masked_attn_status()
        G = out.shape[2] // Hkv
        total = torch.einsum("bsn,nd->bsd", seen.double(), vals.double())
        assert total.abs().max() < 2 ** 24
        ref = torch.where(count > 0, total / count.clamp(min=1), 0.0)
        ref = torch.stack([ref.roll(h // G, -1) for h in range(out.shape[2])], 2)
        tol = ref.abs() * (torch.finfo(dtype).eps / 2 + 2.0 ** -22) + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
        err = (out.double() - ref).abs()
        assert (err <= tol).all(), f"{(err > tol).nonzero()[:4].tolist()} {'single keys' if vals is lone else 'tiles'}"


def _zero(dev, B, Sq, Hq, D, dtype):
    return torch.zeros(B, Sq, Hq, D, device=dev, dtype=dtype)


SCORES = [dict(), dict(softcap=30.0), "slopes", "table"]


def _score(kw, Hq, dev):
    if kw == "slopes":
        return dict(slopes=torch.zeros(Hq, device=dev))
    if kw == "table":
        return dict(bias_table=torch.zeros(Hq, 33, device=dev))
    return kw


@pytest.mark.parametrize("score", SCORES, ids=["plain", "cap", "slopes", "table"])
@pytest.mark.parametrize("B,Sq,Skv,Hq,Hkv,D,dtype", [
    (1, 1, 40000, 2, 2, 64, BF16), (3, 1, 9001, 8, 2, 128, FP16), (4, 1, 4097, 12, 12, 64, BF16), (2, 5, 3000, 8, 4, 256, BF16),
    (2, 17, 2000, 12, 1, 96, FP16), (2, 100, 5000, 4, 4, 128, BF16), (1, 300, 300, 2, 2, 64, FP16), (4, 300, 700, 40, 8, 64, BF16),
    (2, 390, 2600, 40, 40, 128, FP16), (3, 200, 450, 4, 1, 256, FP16),
])
def test_every_key_once(cuda, B, Sq, Skv, Hq, Hkv, D, dtype, score):
    from quantfun2_b200 import attention as A

    q = _zero(cuda, B, Sq, Hq, D, dtype)
    score = _score(score, Hq, cuda)
    g = torch.Generator().manual_seed(Skv)
    lens = torch.randint(max(1, Skv // 3), Skv + 1, (B,), generator=g)
    lens[-1] = Skv
    end = [n - Sq for n in lens.tolist()]
    dlens = lens.to(cuda)
    for window in ((-1, -1), (-1, 0), (Skv // 3, 0), (130, 40)):
        call = lambda k, v, *_: A.masked_attn(q, k, v, window=window, tensor_layout="NHD", **score)  # noqa: E731,B023
        _check(call, _seen(cuda, B, Sq, Skv, window=window), Hkv, D, dtype)
        call = lambda k, v, *_: A.masked_attn(q, k, v, window=window, kv_lens=dlens, q_offset="end", tensor_layout="NHD", **score)  # noqa: E731,B023
        _check(call, _seen(cuda, B, Sq, Skv, window=window, offsets=end, kv_lens=lens.tolist()), Hkv, D, dtype)


@pytest.mark.parametrize("D,dtype,Hq,Hkv", [(64, BF16, 2, 1), (128, BF16, 2, 2)])
def test_every_key_of_the_longest_cache(cuda, D, dtype, Hq, Hkv):
    from quantfun2_b200 import attention as A

    S = 1 << 20
    q = _zero(cuda, 1, 1, Hq, D, dtype)
    for n, window in ((S, (-1, 0)), (S - 77, (-1, 0)), (S - 128, (300, 0)), (S, (S - 129, 0))):
        lens = torch.tensor([n], device=cuda)
        call = lambda k, v, *_: A.masked_attn(q, k, v, window=window, kv_lens=lens, q_offset="end", tensor_layout="NHD")  # noqa: E731,B023
        _check(call, _seen(cuda, 1, 1, S, window=window, offsets=[n - 1], kv_lens=[n]), Hkv, D, dtype)


@pytest.mark.parametrize("B,S,Hq,Hkv,D,dtype", [(3, 260, 4, 2, 64, BF16), (3, 520, 40, 40, 96, FP16), (2, 2500, 24, 8, 128, BF16), (3, 300, 4, 2, 256, BF16)])
def test_every_key_of_documents_and_prefixes(cuda, B, S, Hq, Hkv, D, dtype):
    from quantfun2_b200 import attention as A

    q = _zero(cuda, B, S, Hq, D, dtype)
    g = torch.Generator(device=cuda).manual_seed(S)
    ids = torch.zeros(B, S, dtype=torch.int32, device=cuda)
    for cut in (1, 40, 128, 200, 256, 259):
        ids[:, cut:] += 1
    ids[1, S * 3 // 4:] = -1
    ids[-1] = torch.randint(-1, 4, (S,), device=cuda, generator=g)
    for window in ((-1, -1), (-1, 0), (70, 30)):
        call = lambda k, v, *_: A.masked_attn(q, k, v, window=window, segment_ids=ids, tensor_layout="NHD")  # noqa: E731,B023
        _check(call, _seen(cuda, B, S, S, window=window, q_ids=ids, k_ids=ids), Hkv, D, dtype)
    pre = [0, 129, S // 2][:B]
    dpre = torch.tensor(pre, device=cuda)
    for window in ((-1, 0), (20, 0)):
        call = lambda k, v, *_: A.masked_attn(q, k, v, window=window, prefix_lens=dpre, tensor_layout="NHD")  # noqa: E731,B023
        _check(call, _seen(cuda, B, S, S, window=window, prefix_lens=pre), Hkv, D, dtype)
        call = lambda k, v, *_: A.masked_attn(q, k, v, window=window, prefix_lens=dpre, segment_ids=ids, tensor_layout="NHD")  # noqa: E731,B023
        _check(call, _seen(cuda, B, S, S, window=window, prefix_lens=pre, q_ids=ids, k_ids=ids), Hkv, D, dtype)


@pytest.mark.parametrize("B,Sq,Skv,P,Hq,Hkv,D,dtype", [
    (64, 1, 300, 3001, 6, 2, 96, FP16), (5, 40, 49, 77, 4, 4, 64, BF16), (2, 300, 300, 130, 2, 1, 256, BF16), (130, 1, 20, 16384, 2, 2, 64, BF16),
    (8, 300, 309, 1000, 24, 8, 128, BF16), (3, 1, 5000, 129, 8, 2, 128, BF16)])
def test_every_key_behind_a_shared_prefix(cuda, B, Sq, Skv, P, Hq, Hkv, D, dtype):
    from quantfun2_b200 import attention as A

    q = _zero(cuda, B, Sq, Hq, D, dtype)
    lens = torch.randint(0, Skv + 1, (B,), generator=torch.Generator().manual_seed(P))
    lens[-1] = Skv
    dlens = lens.to(cuda)
    for window in ((-1, 0), (P // 2, 0)):
        call = lambda k, v, pk, pv: A.shared_prefix_attn(q, pk, pv, k, v, window=window, kv_lens=dlens, q_offset=Skv - Sq, tensor_layout="NHD")  # noqa: E731,B023
        _check(call, _seen(cuda, B, Sq, Skv, P, window=window, offsets=[Skv - Sq] * B, kv_lens=lens.tolist()), Hkv, D, dtype, P)


# splits by what each element has to read, decided on the device
UNLIKE = [(16, 1, 4000, 12, 4, 64, BF16, 0), (2, 100, 20000, 12, 4, 64, FP16, 0), (8, 5, 8000, 8, 8, 128, BF16, 0), (4, 1, 20000, 24, 8, 128, BF16, 0),
          (3, 1, 30000, 4, 4, 96, FP16, 0), (2, 5, 9000, 8, 4, 256, BF16, 0), (2, 100, 9000, 4, 4, 128, FP16, 0), (5, 1, 20000, 8, 8, 64, BF16, 700),
          (5, 40, 9000, 2, 2, 128, FP16, 700), (30, 1, 4000, 6, 2, 96, BF16, 700)]


def _unlike(B, Skv):
    lens = torch.randint(0, Skv + 1, (B,), generator=torch.Generator().manual_seed(B))
    lens[0], lens[B // 2] = Skv, 1
    if B > 2:
        lens[1] = 0
    return lens.tolist()


@pytest.mark.parametrize("B,Sq,Skv,Hq,Hkv,D,dtype,P", UNLIKE)
def test_every_key_of_unlike_lengths(cuda, B, Sq, Skv, Hq, Hkv, D, dtype, P):
    from quantfun2_b200 import attention as A

    q = _zero(cuda, B, Sq, Hq, D, dtype)
    for lens in (_unlike(B, Skv), [Skv] * B, [Skv] + [0] * (B - 1), [0] * B):
        dlens, end = torch.tensor(lens, device=cuda), [n - Sq for n in lens]
        for window, score in (((-1, 0), {}), ((-1, 0), dict(softcap=30.0)), ((Skv // 2, 0), {})):
            kw = dict(window=window, kv_lens=dlens, q_offset="end", tensor_layout="NHD", **score)
            call = (lambda k, v, pk, pv: A.shared_prefix_attn(q, pk, pv, k, v, **kw)) if P else (  # noqa: B023
                lambda k, v, pk, pv: A.masked_attn(q, k, v, **kw))  # noqa: B023
            _check(call, _seen(cuda, B, Sq, Skv, P, window=window, offsets=end, kv_lens=lens), Hkv, D, dtype, P)


@pytest.mark.parametrize("B,Sq,Skv,Hq,Hkv,D,dtype,P", UNLIKE)
def test_caches_of_unlike_lengths(cuda, B, Sq, Skv, Hq, Hkv, D, dtype, P):
    """Against the formula, with and without a bias; the bits of a second call."""
    from quantfun2_b200 import attention as A
    from test_gpu_text_attention import _compare, _inputs

    made = _inputs(cuda, B, Sq, Skv, Hq, Hkv, D, dtype, seed=80, P=P)
    (q, k, v), pre = made[:3], made[3:]
    lens = _unlike(B, Skv)
    pick, rows = sorted({0, B // 2, B - 1}), sorted({0, Sq - 1})
    off = [n - Sq for n in lens]
    for more in (dict(), dict(slopes=torch.rand(Hq, device=cuda) * 0.01), dict(softcap=20.0)):
        kw = dict(window=(-1, 0), kv_lens=torch.tensor(lens, device=cuda), q_offset="end", tensor_layout="NHD", **more)
        call = (lambda: A.shared_prefix_attn(q, *pre, k, v, **kw)) if P else (lambda: A.masked_attn(q, k, v, **kw))  # noqa: B023
        out = call()
        ref = dict(prefix_k=pre[0], prefix_v=pre[1]) if P else {}
        _compare(out[pick], q[pick], k[pick], v[pick], rows=rows, window=(-1, 0), kv_lens=[lens[b] for b in pick],
                 offsets=[off[b] for b in pick], **more, **ref)
        assert torch.equal(out, call())
