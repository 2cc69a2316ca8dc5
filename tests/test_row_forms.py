"""The calls of test_gpu_row_forms.py run every form of the row attention's fast kernels, by the dispatch rules as
row_forms.py restates them; where a rule decides over a workspace, the library's own answer agrees."""

import pytest

from taco_amd import hip
from tests import row_forms as forms


def test_every_form_has_a_call():
    for mass in (False, True):
        reached = {forms.form(*s, score_s, mass) for s in forms.SHAPES for score_s in forms.SCORES}
        assert set(forms.FORMS) <= reached, sorted(set(forms.FORMS) - reached)
    reached = {forms.form(b, 1, h, hd, cap, score_s, True) for b, h, hd, cap in forms.ONE_ROW for score_s in forms.SCORES}
    assert set(forms.DECODE_FORMS) <= reached, sorted(set(forms.DECODE_FORMS) - reached)


@pytest.mark.parametrize("shape", forms.SHAPES + [(b, 1, h, hd, cap) for b, h, hd, cap in forms.ONE_ROW] +
                         [(8, 64, 25, 64, 8192), (1, 256, 12, 64, 65_536), (600, 17, 1, 80, 140_000), (64, 1, 12, 64, 8000),
                          (1, 1, 12, 64, 2000), (20, 3, 7, 128, 4097), (2, 5, 2, 20, 5000), (1000, 1, 2, 128, 300), (1000, 1, 2, 128, 900)])
def test_workspaces_follow_the_rules(shape):
    """hs_op_attend_rows_workspace gives the most over a tree and causal rows, a short table and a long one."""
    want = max(forms.workspace(*shape, mass, table) for mass in (False, True) for table in (1, 20_000))
    assert hip.attend_rows_workspace(*shape) == want
