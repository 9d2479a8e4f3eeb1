"""Addresses of the verification operators that are off their type: refused with
a status and a message before any CUDA work (no GPU needed)."""
import pytest

import vspec_b200 as V
from test_verify_ops_abi_cpu import P, _append, _gather, _lp, _refused, _rope, _tree


# (call, argument, bytes its type takes)
ALIGNMENT = [
    (_rope, "d_q", 4), (_rope, "d_k", 4), (_rope, "d_q_out", 4), (_rope, "d_k_out", 4), (_rope, "d_pos", 4),
    (_rope, "d_turns", 8), (_append, "d_k", 4), (_append, "d_v", 4), (_append, "d_slots", 4), (_append, "d_k_scales", 4),
    (_append, "d_v_scales", 4), (_gather, "d_k_scales", 4), (_gather, "d_v_scales", 4), (_gather, "d_page_table", 4),
    (_gather, "d_cu_tokens", 4), (_gather, "d_k_out", 4), (_gather, "d_v_out", 4), (_tree, "d_page_table", 4),
    (_tree, "d_ctx_len", 4), (_tree, "d_cu_q", 4), (_tree, "d_mask", 4), (_lp, "d_allowed", 4), (_lp, "d_tokens", 4),
    (_lp, "d_token_logprobs", 4), (_lp, "d_entropy", 4), (_lp, "d_top_logprobs", 4), (_lp, "d_top_ids", 4)]


@pytest.mark.parametrize("call,name,size", ALIGNMENT)
def test_addresses_off_their_type_are_refused(call, name, size):
    """An address that is no multiple of its values' size would fault on the device."""
    for off in (1, size // 2):
        _refused(call(**{name: P + off}), V.ERR_ARG, "aligned")


@pytest.mark.parametrize("call,names,dtype", [(_rope, ["d_q", "d_k", "d_q_out", "d_k_out"], "dtype"),
                                              (_append, ["d_k", "d_v"], "src_dtype"),
                                              (_gather, ["d_k_out", "d_v_out"], "out_dtype")])
@pytest.mark.parametrize("kind", [V.T_F16, V.T_BF16])
def test_odd_addresses_of_16_bit_values_are_refused(call, names, dtype, kind):
    for name in names:
        _refused(call(**{name: P + 1, dtype: kind}), V.ERR_ARG, "aligned")
