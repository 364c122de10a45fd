"""GPU: bounded waits of the masked attention kernel that run out, without a GPU fault.

qf2_masked_attn_fault_injection shortens every wait to about 2 ms and leaves one key tile of each
block unloaded, a barrier that nothing completes.  The warps that wait on it give up, the others
see it and follow, the copies and products in flight end, tensor memory is freed and the status
word tells the host; the next normal call on the same context gives the bits of the one before."""
import pytest
import torch

from quantfun2_b200 import _lib
from quantfun2_b200._lib import QF2Error

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


# (form, splits; the tile is one that a block has): single tiles twice on an SM, one on an SM, pairs,
# few rows of many splits, by lengths, behind a prefix
CASES = [(4, 300, 700, 40, 8, 64, BF16, 0, 1), (1, 200, 300, 2, 2, 128, FP16, 0, 0), (2, 300, 900, 4, 2, 256, BF16, 0, 0),
         (4, 390, 2600, 24, 8, 128, BF16, 0, 3), (4, 390, 2600, 24, 8, 64, FP16, 0, 0), (1, 1, 9000, 4, 2, 128, BF16, 0, 0),
         (4, 1, 20000, 24, 8, 128, BF16, 0, 1), (16, 1, 4000, 12, 4, 64, FP16, 0, 0)]


@pytest.mark.parametrize("B,Sq,Skv,Hq,Hkv,D,dtype,P,tile,ids", [(*c, ids) for c in CASES for ids in (False, True)] + [
    (30, 1, 300, 6, 2, 96, BF16, 700, 0, False)])
def test_a_wait_that_runs_out_is_reported_and_passes(cuda, B, Sq, Skv, Hq, Hkv, D, dtype, P, tile, ids):
    from quantfun2_b200 import attention as A

    g = torch.Generator(device=cuda).manual_seed(90)
    r = lambda *s: torch.randn(*s, device=cuda, generator=g).to(dtype)  # noqa: E731
    q, k, v, pk, pv = r(B, Sq, Hq, D), r(B, Skv, Hkv, D), r(B, Skv, Hkv, D), r(P, Hkv, D), r(P, Hkv, D)
    lens = torch.full((B,), Skv, device=cuda, dtype=torch.int32)
    kw = dict(window=(-1, 0), kv_lens=lens, q_offset="end", tensor_layout="NHD")
    if ids:
        key = torch.randint(0, 3, (B, Skv), device=cuda, generator=g)
        kw["segment_ids"] = (key[:, -Sq:].contiguous(), key)
    call = (lambda: A.shared_prefix_attn(q, pk, pv, k, v, **kw)) if P else (lambda: A.masked_attn(q, k, v, **kw))
    clean = call()
    A.masked_attn_status()
    lib = _lib.load()
    assert lib.qf2_masked_attn_fault_injection(2000, tile) == 0
    try:
        call()
        with pytest.raises(QF2Error, match="timed out"):
            A.masked_attn_status()
        A.masked_attn_status()                                    # the read cleared it
    finally:
        lib.qf2_masked_attn_fault_injection(0, -1)
    assert torch.equal(call(), clean)
    A.masked_attn_status()
