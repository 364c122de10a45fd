"""CPU: which kernel form and splits the GPU tests of masked attention reach.  The choice follows
from fitted estimates; a change of theirs must not take a form out of the tests unseen."""
import pytest

import test_gpu_text_attention as gpu
import test_gpu_text_keys as keys
from quantfun2_b200 import _lib

SMALL, DEEP, PAIR = 0, 1, 2


def plan(B, Sq, Skv, Hq, Hkv, D, P=0, window=(-1, -1), lens=False, end=False, array=False, prefix=False, ids=0, score=False,
         table=False):
    """The plan of a call; lens, prefix, ids, ...: whether (and of ids in how many words) they are given."""
    a = dict(B=B, Hq=Hq, Hkv=Hkv, Sq=Sq, Skv=Skv, D=D, P=P, left=window[0], right=window[1], kv_lens=lens, prefix_lens=prefix,
             q_offset=Skv - Sq, q_offset_mode=2 if end else 1 if array else 0, q_ids=ids > 0, k_ids=ids > 0, ids_i64=ids == 2,
             slopes=score, bias_table=table)
    out = _lib.i64(*[0] * 8)
    assert _lib.load().qf2_masked_attn_plan(_lib.MASKED_ATTN_ARGS.pack_named(**a), out) == 0
    names = ("form", "heads", "tokens", "splits", "even", "elements", "prefix_splits", "bytes")
    return dict(zip(names, out))


def cases(test):
    """Parameters of a GPU test, from its mark."""
    marks = [m for m in test.pytestmark if m.name == "parametrize"]
    assert len(marks) == 1
    return marks[0].args[1]


def test_tests_of_pairs_reach_pairs():
    for B, Sq, Skv, Hq, Hkv, D, _, window in cases(gpu.test_pairs_of_query_tiles):
        assert plan(B, Sq, Skv, Hq, Hkv, D, window=window)["form"] == PAIR, (B, Sq, Skv, D)
    for D, _ in cases(gpu.test_pairs_with_capped_and_biased_scores):
        for kw in (dict(table=True), dict(score=True), dict(score=True, window=(-1, 0)), dict(score=True, window=(2100, 20))):
            assert plan(3, 500, 2500, 32, 16, D, **kw)["form"] == PAIR, (D, kw)
    for kw in (dict(window=(-1, 0), prefix=True), dict(window=(1800, 0), prefix=True, lens=True, array=True),
               dict(window=(-1, 0), lens=True, end=True), dict(ids=2), dict(ids=2, window=(-1, 0))):
        assert plan(5, 500, 2500, 24, 8, 96, **kw)["form"] == PAIR, kw
    for kw in (dict(lens=True), dict(ids=1), dict(window=(1500, 0))):
        assert plan(4, 500, 2600, 24, 12, 128, **kw)["form"] == PAIR, kw
    for D, _ in cases(gpu.test_pairs_behind_a_shared_prefix):
        for score in (False, True):
            assert plan(5, 500, 509, 24, 8, D, P=2100, window=(-1, 0), lens=True, score=score)["form"] == PAIR, D
    # of those beside them
    assert plan(4, 500, 2500, 24, 8, 128, ids=2)["form"] == PAIR                         # 64-bit ids
    assert plan(2, 500, 2600, 48, 24, 96, score=True, lens=True)["form"] == PAIR         # hidden keys under a cap
    assert plan(3, 500, 2600, 48, 48, 128, array=True, score=True)["form"] == PAIR       # far slopes
    assert plan(2, 2500, 2500, 24, 24, 128, window=(-1, 0))["form"] == PAIR              # outputs over inputs


def test_every_form_meets_every_mask():
    met = set()

    def note(what, **kw):
        p = plan(**kw)
        met.add((p["form"], what))
        if p["splits"] > 1:
            met.add((p["form"], "splits"))
        if p["even"]:
            met.add((p["form"], "even"))
            if kw.get("P"):
                met.add((p["form"], "even behind a prefix"))
        if p["elements"]:
            met.add((p["form"], "prefix items"))
        elif kw.get("P"):
            met.add((p["form"], "prefix walked"))
        if p["heads"] > 1:
            met.add((p["form"], "packed heads"))

    for B, Sq, Hq, Hkv, D, _, causal in cases(gpu.test_dense_and_causal):
        note("dense", B=B, Sq=Sq, Skv=Sq, Hq=Hq, Hkv=Hkv, D=D, window=(-1, 0 if causal else -1))
    for B, S, Hq, Hkv, D, _, window in cases(gpu.test_two_tile_grids):
        note("dense", B=B, Sq=S, Skv=S, Hq=Hq, Hkv=Hkv, D=D, window=window)
    for B, Sq, Skv, Hq, Hkv, D, _ in cases(gpu.test_few_tokens_on_caches):
        for score, table in ((False, False), (True, False), (False, True)):
            note("score" if score else "table" if table else "lengths", B=B, Sq=Sq, Skv=Skv, Hq=Hq, Hkv=Hkv, D=D,
                 window=(-1, 0), lens=True, end=True, score=score, table=table)
    for B, S, P, Hq, Hkv, D, _ in cases(gpu.test_shared_prefix):
        for score, table in ((False, False), (True, False), (False, True)):
            note("prefix", B=B, Sq=S, Skv=S + 9, P=P, Hq=Hq, Hkv=Hkv, D=D, window=(-1, 0), lens=True, score=score, table=table)
    for Hq, two in ((2, False), (80, True)):
        for D in (64, 128):
            note("table", B=2, Sq=290, Skv=290, Hq=Hq, Hkv=Hq // 2, D=D, table=True)
            note("score", B=2, Sq=290, Skv=290, Hq=Hq, Hkv=Hq // 2, D=D, score=True, window=(-1, 0))
    for B, Sq, Skv, Hq, Hkv, D, _ in cases(gpu.test_ids_in_64_bits):
        note("ids", B=B, Sq=Sq, Skv=Skv, Hq=Hq, Hkv=Hkv, D=D, ids=2)
    for B, S, Hq, Hkv, D, _ in cases(keys.test_every_key_of_documents_and_prefixes):
        note("ids", B=B, Sq=S, Skv=S, Hq=Hq, Hkv=Hkv, D=D, ids=1, window=(-1, 0))
        note("prefix lengths", B=B, Sq=S, Skv=S, Hq=Hq, Hkv=Hkv, D=D, prefix=True, window=(-1, 0))
    for B, Sq, Skv, Hq, Hkv, D, _, P in keys.UNLIKE:
        note("lengths", B=B, Sq=Sq, Skv=Skv, P=P, Hq=Hq, Hkv=Hkv, D=D, window=(-1, 0), lens=True, end=True)
    for B, Sq, Skv, P, Hq, Hkv, D, _ in cases(keys.test_every_key_behind_a_shared_prefix):
        note("prefix", B=B, Sq=Sq, Skv=Skv, P=P, Hq=Hq, Hkv=Hkv, D=D, lens=True, window=(-1, 0))
    for D, _ in cases(gpu.test_pairs_behind_a_shared_prefix):
        note("prefix", B=5, Sq=500, Skv=509, P=2100, Hq=24, Hkv=8, D=D, lens=True, window=(-1, 0))

    for form in (SMALL, DEEP):
        for what in ("dense", "score", "table", "ids", "prefix lengths", "packed heads", "splits", "even", "prefix walked"):
            assert (form, what) in met, (form, what)
    assert (SMALL, "prefix items") in met and (SMALL, "even behind a prefix") in met
    for what in ("ids", "prefix lengths", "prefix walked"):
        assert (PAIR, what) in met, what


def test_plans_of_common_calls():
    p = plan(1, 16384, 16384, 24, 8, 128, window=(-1, 0))
    assert (p["form"], p["heads"], p["splits"], p["bytes"]) == (PAIR, 1, 1, 0)
    p = plan(4, 1, 32768, 24, 8, 128, window=(-1, 0), lens=True, end=True)
    assert p["heads"] == 3 and p["even"] > 0 and p["bytes"] > 0
    p = plan(64, 1, 512, 24, 8, 128, P=16384, window=(-1, 0), lens=True, end=True)
    assert p["elements"] == 42 and p["prefix_splits"] > 1                    # 42 x 3 rows of a tile
    for ids in (0, 1, 2):                                                    # never more than the sizes' workspace
        p = plan(2, 300, 5000, 12, 4, 128, ids=ids, window=(70, 0))
        assert p["bytes"] <= _lib.load().qf2_masked_attn_workspace_bytes(2, 12, 4, 300, 5000, 0, 128, ids)


@pytest.mark.parametrize("kw,status", [(dict(D=80), -1), (dict(Hq=3, Hkv=2), -1), (dict(Sq=-1), -1)])
def test_plan_refuses_what_the_call_refuses(kw, status):
    a = dict(B=1, Hq=2, Hkv=2, Sq=4, Skv=4, D=64, left=-1, right=-1)
    a.update(kw)
    out = _lib.i64(*[0] * 8)
    lib = _lib.load()
    assert lib.qf2_masked_attn_plan(_lib.MASKED_ATTN_ARGS.pack_named(**a), out) == status
    assert lib.qf2_masked_attn_plan(None, out) == -8
