"""States that lack a tensor are refused by its name, also where the moments alone are asked for."""
import pytest
import torch

import modulated_deform_conv as mdc


@pytest.mark.parametrize("missing", ["exp_avg", "exp_avg_sq", "step", "exp_avg_scale", "exp_avg_sq_scale"])
def test_moments_of_a_state_without_one(missing):
    state = mdc.adamw_state([torch.zeros(5)], 8)
    del state[missing]
    with pytest.raises(RuntimeError, match=f"the state has no '{missing}'"):
        mdc.adamw_moments(state)
