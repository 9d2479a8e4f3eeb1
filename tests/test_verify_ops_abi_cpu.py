"""Refusals of the verification operators: every bad argument returns a status
and a message before any CUDA work (no GPU needed)."""
import ctypes

import numpy as np
import pytest

import vspec_b200 as V

P = 1 << 12   # a well aligned address that is never followed


def _refused(rc, status, *words):
    assert rc == status
    for w in words:
        assert w in V.last_error()


def _rope(**kw):
    a = dict(d_q=P, d_k=P, d_q_out=P, d_k_out=P, d_pos=P, d_turns=P, tokens=1, num_q_heads=2, num_k_heads=1,
             head_dim=64, rot_dim=64, q_stride=0, k_stride=0, q_out_stride=0, k_out_stride=0, attn_factor=1.0, dtype=0,
             flags=0)
    a.update(kw)
    return V.lib.vspec_b200_rope(ctypes.byref(V.RopeArgs(**a)), None)


@pytest.mark.parametrize("kw,word", [
    (dict(d_q=None), "NULL"), (dict(d_pos=None), "NULL"), (dict(d_turns=None), "NULL"), (dict(d_k_out=None), "together"),
    (dict(dtype=3), "dtype"), (dict(flags=4), "flags"), (dict(rot_dim=63), "rot_dim"), (dict(rot_dim=66), "rot_dim"),
    (dict(rot_dim=0), "rot_dim"), (dict(head_dim=1024), "head_dim"), (dict(num_q_heads=0), "zero"),
    (dict(num_k_heads=0), "zero"), (dict(q_stride=64), "stride"), (dict(k_out_stride=8), "stride"),
    (dict(q_stride=256), "in place"), (dict(num_q_heads=1 << 20), "heads"), (dict(tokens=1 << 33), "tokens")])
def test_rope_refusals(kw, word):
    _refused(_rope(**kw), V.ERR_ARG, word)


def test_rope_of_no_tokens_is_nothing():
    assert _rope(tokens=0) == V.OK


@pytest.mark.parametrize("args,word", [((63, 1e6), "rot_dim"), ((0, 1e6), "rot_dim"), ((64, 1.0), "theta"),
                                       ((64, float("inf")), "theta"), ((64, 1e6, 7), "scaling"),
                                       ((64, 1e6, V.ROPE_LINEAR, 0.5), "factor"),
                                       ((64, 1e6, V.ROPE_YARN, 2.0, 0.0), "original_ctx"),
                                       ((64, 1e6, V.ROPE_YARN, 2.0, 4096, 1.0, 2.0), "beta")])
def test_rope_turns_refusals(args, word):
    with pytest.raises(V.VspecB200Error, match=word):
        V.rope_turns(*args)


def test_rope_turns_plain_values():
    turns, mult = V.rope_turns(4, 100.0)
    assert mult == 1.0
    assert np.allclose(turns.astype(np.float64) / 2.0 ** 64 * 2 * np.pi, [1.0, 0.1], rtol=1e-14)


def _append(**kw):
    a = dict(d_k=P, d_v=P, d_slots=None, rows=1, num_kv_heads=1, head_dim=64, k_stride=0, v_stride=0, pool_rows=4,
             d_k_codes=P, d_v_codes=P, d_k_scales=P, d_v_scales=P, src_dtype=0, kv_dtype=V.KV_FP8)
    a.update(kw)
    return V.lib.vspec_b200_kv_quant_append(ctypes.byref(V.KvQuantArgs(**a)), None)


@pytest.mark.parametrize("kw,status,word", [
    (dict(d_k=None), 1, "NULL"), (dict(d_v_scales=None), 1, "NULL"), (dict(src_dtype=9), 1, "src_dtype"),
    (dict(kv_dtype=V.KV_F16), 1, "kv_dtype"), (dict(kv_dtype=V.KV_INT3), 1, "kv_dtype"), (dict(head_dim=0), 1, "zero"),
    (dict(pool_rows=0), 1, "zero"), (dict(head_dim=513), 3, "head_dim"), (dict(k_stride=32), 1, "stride"),
    (dict(rows=1 << 33), 1, "rows")])
def test_kv_append_refusals(kw, status, word):
    _refused(_append(**kw), status, word)


def _gather(**kw):
    a = dict(d_k_codes=P, d_v_codes=P, d_k_scales=P, d_v_scales=P, d_page_table=P, d_cu_tokens=P, batch=1,
             total_tokens=1, num_kv_heads=1, head_dim=64, page_tokens=16, max_pages_per_seq=1, num_pages=1, d_k_out=P,
             d_v_out=P, out_dtype=0, kv_dtype=V.KV_INT8)
    a.update(kw)
    return V.lib.vspec_b200_kv_quant_gather(ctypes.byref(V.KvGatherArgs(**a)), None)


@pytest.mark.parametrize("kw,word", [
    (dict(d_cu_tokens=None), "NULL"), (dict(d_k_out=None), "NULL"), (dict(out_dtype=-1), "out_dtype"),
    (dict(kv_dtype=V.KV_F32), "kv_dtype"), (dict(batch=0), "zero"), (dict(page_tokens=0), "zero"),
    (dict(total_tokens=1 << 32), "large"), (dict(head_dim=1000), "large")])
def test_kv_gather_refusals(kw, word):
    _refused(_gather(**kw), V.ERR_ARG, word)


def _tree(**kw):
    a = dict(d_q=P, d_k_pages=P, d_v_pages=P, d_k_scales=P, d_v_scales=P, d_page_table=P, d_ctx_len=P, d_cu_q=P,
             d_mask=P, d_out=P, batch=1, total_q=4, max_q=4, num_q_heads=4, num_kv_heads=2, head_dim=128,
             page_tokens=16, max_pages_per_seq=4, num_pages=8, max_ctx=64, mask_words=1, q_stride=0, scale=0.1,
             q_dtype=0, kv_dtype=V.KV_FP8, d_workspace=None, workspace_bytes=0)
    a.update(kw)
    return V.lib.vspec_b200_tree_attention(ctypes.byref(V.TreeAttnArgs(**a)), None)


@pytest.mark.parametrize("kw,status,word", [
    (dict(d_q=None), 1, "NULL"), (dict(d_k_scales=None), 1, "NULL"), (dict(d_ctx_len=None), 1, "NULL"),
    (dict(q_dtype=5), 1, "q_dtype"), (dict(kv_dtype=V.KV_F32), 1, "kv_dtype"), (dict(kv_dtype=V.KV_INT3), 1, "kv_dtype"),
    (dict(max_q=0), 1, "zero"), (dict(num_pages=0), 1, "zero"), (dict(num_q_heads=5), 1, "multiple"),
    (dict(head_dim=72), 3, "head_dim"), (dict(head_dim=272), 3, "head_dim"),
    (dict(head_dim=60, kv_dtype=V.KV_F16), 3, "head_dim"), (dict(max_ctx=65), 1, "exceeds"),
    (dict(max_q=33, total_q=33), 1, "mask_words"), (dict(d_cu_q=None, total_q=5), 1, "total_q"),
    (dict(q_stride=256), 1, "q_stride"), (dict(q_stride=516), 1, "q_stride"), (dict(d_out=P + 4), 1, "aligned"),
    (dict(d_v_pages=P + 8), 1, "aligned"), (dict(num_pages=1 << 28), 1, "large"), (dict(batch=1 << 17), 1, "large")])
def test_tree_attention_refusals(kw, status, word):
    _refused(_tree(**kw), status, word)


def test_tree_attention_of_no_tokens_is_nothing():
    assert _tree(total_q=0) == V.OK


def test_tree_attention_workspace_of_bad_sizes_is_zero():
    ws = V.lib.vspec_b200_tree_attention_workspace_bytes
    assert ws(0, 1, 1, 1, 1, 64, 64) == 0
    assert ws(1, 1, 1, 3, 2, 64, 64) == 0
    assert ws(1, 1, 1, 1, 1, 64, 0) == 0


def _lp(**kw):
    a = dict(d_logits=P, d_allowed=None, d_tokens=P, d_token_logprobs=P, d_entropy=P, d_top_logprobs=P, d_top_ids=P,
             rows=1, vocab=100, row_stride=0, num_tokens=1, top_k=5, inv_temperature=1.0, dtype=0, d_workspace=None,
             workspace_bytes=0)
    a.update(kw)
    return V.lib.vspec_b200_logprobs(ctypes.byref(V.LogprobsArgs(**a)), None)


@pytest.mark.parametrize("kw,status,word", [
    (dict(d_logits=None), 1, "NULL"), (dict(dtype=4), 1, "dtype"), (dict(vocab=0), 1, "vocab"),
    (dict(vocab=1 << 31), 1, "vocab"), (dict(row_stride=99), 1, "row_stride"), (dict(d_tokens=None), 1, "num_tokens"),
    (dict(d_top_ids=None), 1, "top_k"), (dict(top_k=33), 3, "top_k"), (dict(inv_temperature=0.0), 1, "inv_temperature"),
    (dict(inv_temperature=-1.0), 1, "inv_temperature"), (dict(inv_temperature=float("nan")), 1, "inv_temperature"),
    (dict(inv_temperature=float("inf")), 1, "inv_temperature"), (dict(rows=70000), 3, "rows"),
    (dict(num_tokens=0, top_k=0, d_entropy=None), 1, "no output"), (dict(d_logits=P + 2), 1, "aligned")])
def test_logprobs_refusals(kw, status, word):
    _refused(_lp(**kw), status, word)


def test_logprobs_of_no_rows_is_nothing():
    assert _lp(rows=0) == V.OK


@pytest.mark.parametrize("name", ["rope", "kv_quant_append", "kv_quant_gather", "tree_attention", "logprobs"])
def test_null_args(name):
    _refused(getattr(V.lib, f"vspec_b200_{name}")(None, None), V.ERR_ARG, "NULL")
