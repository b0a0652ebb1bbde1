"""Windows with first tokens that stay visible: configuration, rings, step tables, and what the entry points refuse (no GPU)."""
import ctypes as C

import pytest
import torch

from msa_b200.cache import DecodeStep, PackedStep, RingSpec, SequenceStateCache, window_of
from msa_b200.hybrid_config import GroupedAttentionSpec, HybridConfig, LatentAttentionSpec
from tests import hybrid_util as U


def spec(window, first, **kw):
    m = U.attention(4, 2, 16, 8, window, 8, 3, **kw)
    m["mask"]["first"] = first
    return m


def test_configuration_reads_the_first_tokens():
    s = GroupedAttentionSpec.parse(spec(17, 4))
    assert (s.window, s.first, s.span) == (17, 4, (17, 4))
    s = GroupedAttentionSpec.parse(U.attention(4, 2, 16, 8, 17, 8, 3))
    assert (s.first, s.span) == (0, 17)
    assert GroupedAttentionSpec.parse(spec(None, 4)).span is None          # everything is visible anyhow
    assert GroupedAttentionSpec.parse(spec(17, None)).span == 17
    with pytest.raises(ValueError, match="first"):
        GroupedAttentionSpec.parse(spec(17, -1))
    m = U.latent(2, 8, 4, 8, 16, 9)
    m["mask"]["first"] = 2
    with pytest.raises(ValueError, match="first"):
        LatentAttentionSpec.parse(m)


def test_windows_name_size_and_first_tokens():
    cfg = U.parallel(40, 50, [U.layer("attention", spec(17, 4), None), U.layer("attention", spec(17, 0), None), U.layer("attention", spec(17, 4), None),
                              U.layer("attention", spec(None, 4), None)])
    assert HybridConfig.parse(cfg).windows == ((17, 4), 17, None)


@pytest.mark.parametrize("key,max_len,want", [(8, 50, (8, 0)), (8, 8, (8, 0)), (8, 5, (5, 0)), (None, 50, (50, 0)), ((8, 3), 50, (8, 3)), ((8, 3), 12, (8, 3)),
                                              ((8, 3), 11, (11, 0)), ((8, 3), 2, (2, 0)), ((1, 60), 50, (50, 0)), ((2 ** 31 - 1, 2 ** 31 - 1), 50, (50, 0))])
def test_a_cache_that_holds_all_that_is_seen_has_one_window(key, max_len, want):
    assert window_of(key, max_len) == want


def test_rings_hold_the_first_rows_beside_the_window():
    c = SequenceStateCache([RingSpec(6, 8, first=3), RingSpec(6, 8), RingSpec(6, None, first=3), RingSpec(6, 48, first=3)], 2, 50, "cpu", torch.float32)
    assert [c.ring[i].shape[1] for i in range(4)] == [11, 8, 50, 50]
    for kw in (dict(first=-1), dict(window=0), dict(window=-3)):
        with pytest.raises(ValueError):
            RingSpec(**{**dict(width=6, window=8), **kw})


def test_contexts_begin_with_the_first_rows_and_the_window():
    c = SequenceStateCache([RingSpec(6, 8, first=3)], 4, 50, "cpu", torch.float32)
    for s, n in (("a", 20), ("b", 10), ("c", 9), ("d", 0)):
        c.acquire(s)
        c.advance(s, n)
    step = PackedStep([(s, [1, 2], []) for s in "abcd"], c, ((8, 3), 8))
    view = step.views[8, 3]
    assert (view.window, view.first) == (8, 3)
    assert view.old_off.tolist() == [0, 10, 20, 29, 29]        # 3 first rows and 7 of the window, or all there are
    assert view.ctx_off.tolist() == [0, 12, 24, 35, 37] and (view.n_ctx, view.n_old) == (37, 29)
    assert (step.views[8].window, step.views[8].first) == (8, 0) and step.views[8].old_off.tolist() == [0, 7, 14, 21, 21]
    d = DecodeStep(2, c, ((8, 3), 8, (60, 1)))
    assert [(d.views[k].window, d.views[k].first) for k in ((8, 3), 8, (60, 1))] == [(8, 3), (8, 0), (50, 0)]


def test_entry_points_refuse_rings_without_room():
    """Checked before anything is launched or read: the pointers here lead nowhere."""
    from msa_b200 import _cabi_lm as A
    lib, p = A.lib(), 1 << 12
    refused = lambda rc: rc != 0 and b"first tokens" in lib.msa_last_error()
    group = A.GroupArgs(proj=p, proj_stride=96, conv_w=p, inv_freq=p, conv_state=p, q_out=p, ring=p, ctx=p, pos=p, tok_seq=p, slot=p, start=p, cu=p, ctx_off=p,
                        old_off=p, ring_rows=10, heads=4, kv_heads=2, dim=16, vdim=16, rot=8, taps=3, q_pitch=16, k_pitch=16, v_pitch=16, n_tok=0, n_seq=0,
                        n_decode=0, n_old=0, window=8, dtype=A.dtype_code(torch.bfloat16))
    attn = A.AttnArgs(qa=p, qa_row=64, qa_head=16, ka=p, ka_row=64, ka_head=16, v=p, v_row=64, v_head=16, out=p, out_row=64, out_head=16, slot=p, start=p, cu=p,
                      ring_rows=10, group=2, seq0=0, seq1=0, max_len=0, heads=4, da=64, db=0, dv=64, window=8, qa_dtype=A.dtype_code(torch.bfloat16),
                      out_dtype=A.dtype_code(torch.bfloat16), dtype=A.dtype_code(torch.bfloat16), scale=0.1)
    for first, bad in ((0, False), (2, False), (3, True), (-1, True), (2 ** 31 - 1, True)):
        assert refused(lib.msa_lm_group_prep_first(C.byref(group), first, None)) == bad
        assert refused(lib.msa_lm_window_attn_first(C.byref(attn), first, None)) == bad
        assert refused(lib.msa_lm_ring_store_first(p, 64, p, p, p, p, 0, 0, 0, 8, first, p, 10, 1, None)) == bad
        assert refused(lib.msa_lm_group_decode_first(p, 64, p, 10, p, p, 0, 4, 2, 64, 64, 8, first, 1, 0.1, 0, None, 0, p, 256, None, None, None)) == bad
    attn.ring_rows, attn.ctx_off, attn.out_head = 0, p, 64
    for first, bad in ((3, False), (-1, True), (2 ** 31 - 8, True)):
        assert refused(lib.msa_lm_window_attn_tc_first(C.byref(attn), first, 0, 0, 0, p, None)) == bad
