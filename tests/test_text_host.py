"""CPU: frequencies, argument checks and work plans of the text-side operators."""
import ctypes
import math

import pytest
import torch

from quantfun2_b200 import _lib
from quantfun2_b200._lib import QF2Error


def test_rotary_frequencies():
    from quantfun2_b200.kernels import rotary_inv_freq

    r = 64
    f = rotary_inv_freq(r, base=500.0)
    ref = torch.tensor([500.0 ** (-2 * p / r) for p in range(r // 2)], dtype=torch.float64)
    assert f.dtype == torch.float64 and torch.allclose(f, ref, rtol=1e-14, atol=0)
    assert torch.allclose(rotary_inv_freq(r, scaling="linear", factor=4.0), rotary_inv_freq(r) / 4, rtol=1e-14, atol=0)
    ntk = rotary_inv_freq(r, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and math.isclose(ntk[-1].item(), rotary_inv_freq(r)[-1].item() / 4, rel_tol=1e-12)
    plain, parts = rotary_inv_freq(r), rotary_inv_freq(r, scaling="by_parts", factor=4.0, original_length=4096)
    for p in range(r // 2):
        turns = 4096 * plain[p].item() / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - 1.0) / 31.0))
        assert math.isclose(parts[p].item(), plain[p].item() * (keep + (1 - keep) / 4), rel_tol=1e-12)
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, base=0.0),
                dict(rotary_dim=8, scaling="linear", factor=-1.0),
                dict(rotary_dim=8, scaling="by_parts", beta_fast=1.0, beta_slow=1.0)):
        with pytest.raises(QF2Error):
            rotary_inv_freq(**bad)


def test_ops_refuse_host_tensors():
    from quantfun2_b200 import attention, kernels

    x = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(QF2Error):
        kernels.rotary_apply(x, None, torch.arange(2), kernels.rotary_inv_freq(64))
    with pytest.raises(QF2Error):
        attention.masked_attn(x, x, x)
    with pytest.raises(QF2Error):
        attention.shared_prefix_attn(x, None, None, x, x)


def _call(**kw):
    """qf2_masked_attn with aligned dummy pointers: every refusal below comes before a launch."""
    a = dict(B=1, Hq=2, Hkv=2, Sq=4, Skv=4, D=64, dtype=_lib.QF2_BF16, sm_scale=0.1, q=1024, k=1024, v=1024, out=1024,
             left=-1, right=-1)
    stride = kw.pop("stride", 64)
    a.update({f"{t}_strides": (stride,) * 3 for t in ("q", "k", "v", "out")}, prefix_k_strides=(stride,) * 2,
             prefix_v_strides=(stride,) * 2)
    a.update(kw)
    return _lib.load().qf2_masked_attn(_lib.MASKED_ATTN_ARGS.pack_named(**a))


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=_lib.QF2_F32), -2), (dict(D=80), -1), (dict(Hq=3), -1), (dict(Hkv=0), -1), (dict(Sq=-1), -1),
    (dict(B=70000), -1), (dict(Skv=(1 << 20) + 1), -1), (dict(Skv=1 << 20, P=1), -1), (dict(q=None), -8), (dict(k=None), -8),
    (dict(out=None), -8), (dict(P=4), -8), (dict(q_ids=1024), -8), (dict(k_ids=1024), -8), (dict(q_offset_mode=3), -8),
    (dict(q_offset_mode=1), -8), (dict(slopes=1024, bias_table=1024), -8), (dict(bias_table=1024, bias_reach=1025), -1),
    (dict(softcap=-1.0), -8), (dict(softcap=math.nan), -8), (dict(sm_scale=0.0), -8), (dict(sm_scale=math.inf), -8),
    (dict(q=1032), -5), (dict(v=1032), -5), (dict(stride=60), -5), (dict(stride=0), -5),
    (dict(q_ids=1024, k_ids=1024), -6), (dict(q_ids=1024, k_ids=1024, prefix_k=1024, prefix_v=1024, P=4), -8),
])
def test_attention_refusals_without_device(kw, status):
    assert _call(**kw) == status


def test_empty_batches_return_at_once():
    assert _call(B=0, q=None) == 0 and _call(Sq=0) == 0


def test_workspace_plans():
    ws = _lib.load().qf2_masked_attn_workspace_bytes
    # long queries: no split; ids: a padded copy of the keys', and one run of keys per query
    assert ws(1, 24, 8, 16384, 16384, 0, 128, 0) == 0
    assert ws(1, 24, 8, 16384, 16384, 0, 128, 1) >= 16384 * 4 + 16384 * 8
    # single tokens on a long cache are split: fp32 rows and (max, sum) pairs of each split
    one = ws(1, 8, 8, 1, 65536, 0, 128, 0)
    assert one > 0 and (one - 0) % 256 == 0
    assert ws(1, 8, 8, 1, 100, 0, 128, 0) == 0                     # one key tile: nothing to split
    assert ws(64, 24, 8, 1, 512, 16384, 128, 0) > 0                 # prefix items have partial rows
    assert ws(1, 24, 7, 1, 1, 0, 128, 0) == -1


def test_rotary_refusals_without_device():
    lib = _lib.load()

    def call(**kw):
        a = dict(xq=1024, xq_out=1024, positions=1024, inv_freq=1024, xq_strides=(64,) * 3, xq_out_strides=(64,) * 3,
                 pos_strides=(0, 1), pos_is_i64=1, B=1, S=1, Hq=1, Hk=0, D=64, rotary_dim=64, dtype=_lib.QF2_BF16, gain=1.0)
        a.update(kw)
        return lib.qf2_rotary_apply(_lib.ROTARY_ARGS.pack_named(**a))

    assert call(dtype=3) == -2 and call(layout=2) == -8 and call(rotary_dim=63) == -1 and call(rotary_dim=66) == -1
    assert call(rotary_dim=0) == -1 and call(D=2048) == -1 and call(B=-1) == -1
    assert call(Hk=1) == -8 and call(xq=None) == -8 and call(positions=None) == -8 and call(inv_freq=None) == -8
    assert call(B=0) == 0 and call(Hq=0) == 0 and call(S=0, positions=None) == 0
    assert lib.qf2_rotary_apply(None) == -8 and lib.qf2_masked_attn(None) == -8


def test_argument_structs_match_the_header():
    """The packed fields, in order, are the header's struct fields."""
    import re
    from pathlib import Path

    text = (Path(__file__).resolve().parent.parent / "include" / "qf2b200.h").read_text()
    for name, args in (("qf2_rotary_args", _lib.ROTARY_ARGS), ("qf2_masked_attn_args", _lib.MASKED_ATTN_ARGS)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields = []
        for decl in body.split(";"):
            if not decl.strip():
                continue
            m = re.match(r"\s*((?:const )?(?:void|int64_t|int32_t|float|double|qf2_stream_t))\s*(\*?)\s*(.*)", decl, re.S)
            base, star, names = m.group(1), m.group(2), m.group(3)
            assert star or base in ("int64_t", "double", "qf2_stream_t"), decl      # 8 bytes each
            for nm in names.split(","):
                arr = re.match(r"\s*(\w+)(?:\[(\d+)\])?", nm)
                fields.append((arr.group(1), int(arr.group(2) or 1), "d" if base == "double" and not star else "q"))
        assert fields == [tuple(f) for f in args.fields]


def test_lengths_and_positions_beyond_32_bits_stay_far():
    from quantfun2_b200.attention import _int32

    x = torch.tensor([2 ** 32 + 3, 2 ** 31, 2 ** 40, -2 ** 40, -1, 7, 2 ** 31 - 1, -2 ** 31])
    got = _int32(x, (8,), "kv_lens", x.device)
    assert got.dtype == torch.int32
    assert got.tolist() == [min(max(n, -2 ** 31), 2 ** 31 - 1) for n in x.tolist()]


def test_workspace_of_64_bit_ids():
    ws = _lib.load().qf2_masked_attn_workspace_bytes
    one, two = ws(2, 24, 8, 4096, 4096, 0, 128, 1), ws(2, 24, 8, 4096, 4096, 0, 128, 2)
    assert two == one + 2 * 4096 * 4                                # the high words of the copy
    assert ws(2, 24, 8, 4096, 4096, 0, 128, 3) == -8 and ws(2, 24, 8, 4096, 4096, 0, 128, -1) == -8
    assert _call(q_ids=1024, k_ids=1024, ids_i64=1) == -6


def test_scales_beyond_fp32_are_refused():
    assert _call(sm_scale=3e38) == -8 and _call(sm_scale=2.4e38, softcap=1.0) == -8
    assert _call(sm_scale=1e-300, B=0) == 0


def test_overlap_of_views():
    """Against the elements themselves, on views of one buffer."""
    import random

    from quantfun2_b200._lib import overlap, overlaps_itself

    def places(t):
        p = torch.zeros(t.shape, dtype=torch.int64) + t.storage_offset()
        for d, (n, s) in enumerate(zip(t.shape, t.stride())):
            p = p + (torch.arange(n) * s).view([-1] + [1] * (t.dim() - d - 1))
        return p.flatten().tolist()

    joint = torch.zeros(2, 50, 8, 64)
    q, k, v = joint[:, :, :5], joint[:, :, 5:7], joint[:, :, 7:]
    assert not overlap(q, k) and not overlap(k, q) and not overlap(q, v) and not overlaps_itself(q)
    assert overlap(q, q) and overlap(joint, k) and overlap(q[:, 3:], q[:, :4]) and not overlap(q[:, 4:], q[:, :4])
    hnd = torch.zeros(2, 8, 50, 64).transpose(1, 2)
    assert not overlap(hnd[:, :, :3], hnd[:, :, 3:]) and overlap(hnd[:, :, :4], hnd[:, :, 3:])
    assert not overlap(joint[..., :32], joint[..., 32:]) and overlap(joint[..., :33], joint[..., 32:])
    assert overlaps_itself(torch.zeros(1, 3).expand(4, 3)) and overlaps_itself(torch.zeros(9).as_strided((3, 4), (2, 1)))
    assert not overlap(torch.zeros(4), torch.zeros(4)) and not overlap(joint[:0], joint)
    rng = random.Random(0)
    buf = torch.zeros(400)
    told = 0
    for _ in range(3000):
        def view():
            dims = [rng.randint(1, 4) for _ in range(3)]
            strides = [rng.choice([0, 1, 2, 4, 8, 12, 24, 48]) for _ in range(3)]
            return buf.as_strided(dims, strides, rng.randint(0, 20))
        a, b = view(), view()
        pa, pb = places(a), places(b)
        if set(pa) & set(pb):
            assert overlap(a, b)
        told += not overlap(a, b)
        if len(set(pa)) < len(pa):
            assert overlaps_itself(a)
    assert told > 100


def test_rotary_in_place_refuses_shared_memory():
    from quantfun2_b200 import kernels

    x = torch.zeros(1, 4, 6, 64)
    pos, f = torch.arange(4), kernels.rotary_inv_freq(64)
    for xq, xk in ((x, x), (x, x[:, :, 2:4]), (x[:, :, :3], x[:, :, 2:]), (x.as_strided((1, 4, 6, 64), (0, 320, 64, 1)), None),
                   (x[:, :, :2], x[:, :1, 2:3].expand(1, 4, 1, 64))):
        with pytest.raises(QF2Error, match="share memory"):
            kernels.rotary_apply_(xq, xk, pos, f)
    with pytest.raises(QF2Error, match="CUDA"):                     # slices side by side come as far as the device
        kernels.rotary_apply_(x[:, :, :4], x[:, :, 4:], pos, f)


def test_derivatives_are_noticed():
    from torch.autograd import forward_ad

    from quantfun2_b200._lib import wants_derivative

    x, w = torch.zeros(3), torch.zeros(3, requires_grad=True)
    assert wants_derivative(x, None, w) and not wants_derivative(x, None)
    with torch.no_grad():
        assert not wants_derivative(w)
        with forward_ad.dual_level():
            d = forward_ad.make_dual(torch.zeros(3), torch.ones(3))
            assert wants_derivative(x, d) and wants_derivative(d * 2) and not wants_derivative(x, None)
    assert not wants_derivative(x)
