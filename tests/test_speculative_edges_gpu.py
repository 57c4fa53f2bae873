"""Where the operators that verify drafted tokens went wrong once, or are easily got wrong, against the plain references in 64 bits."""

import math

import pytest
import torch

from plain import speculative as plain
from test_speculative_gpu import DEV, K, drafts, i32, verify_both

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ verification
@pytest.mark.parametrize("dense", [False, True])
@pytest.mark.parametrize("what", [-math.inf, math.nan])
def test_verify_accepts_nothing_on_a_row_without_logits(what, dense):
    """A row of which no logit is above -inf says nothing, not that word 0 is the best: a drafted word 0 behind it is not accepted, by a
    greedy request either. (Rows 1 and 4 are behind the root; row 6 is a root's.)"""
    args, q = drafts([3, 3, 2], 3000, seed=2, branch=1, dense=dense)
    for row in (1, 4, 6):
        args["logits"][row] = what
    for node in (1, 4):
        args["tokens"][node] = int(args["logits"][node - 1].argmax())
    for node in (2, 5, 7):
        args["tokens"][node] = 0
    for temp in (None, torch.zeros(3), torch.tensor([0.0, 0.9, 0.0]), torch.tensor([0.9, 0.0, 0.9])):
        got, want = verify_both(args, 3, 2, temp, q)
        assert got == want
        assert got[2] == [[0, -1, -1], [0, -1, -1], 1]
        for s in range(2):
            if temp is None or temp[s] == 0:
                assert got[s][2] == 2 and got[s][0][1] == 0
    K().check_device_errors()
