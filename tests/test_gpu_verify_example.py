"""The verification example end to end: the tree accepts what decoding token by
token says, with the same log probabilities and the same committed cache."""
import os
import sys

import pytest

from gpu_util import torch_cuda

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples"))

pytestmark = pytest.mark.gpu

# The linears agree within 1e-3 of a row's largest value whatever the number of rows (logits of about 4), so two log
# probabilities within a few of those; a K or V value that lands on the other side of a rounding step of its fp8 code
# moves by 2^-3 of itself at most.
LOGPROB = 2e-2
CACHE = 2.0 ** -3


@pytest.mark.parametrize("seed", [0, 1])
def test_tree_verification_matches_token_by_token(seed):
    torch_cuda()
    import tree_verify
    worst, drift = tree_verify.main(seed)
    assert worst <= LOGPROB and drift <= CACHE
