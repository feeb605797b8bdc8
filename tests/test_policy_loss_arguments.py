"""Coefficients of the policy loss that fp32 does not hold (no GPU needed)."""

import pytest
import torch


@pytest.mark.parametrize("kl_coef", [1e39, -1e300])
def test_kl_coefficients_beyond_fp32_are_refused(kl_coef):
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_policy_loss

    x, w, t, f = torch.zeros(4, 64), torch.zeros(100, 64), torch.zeros(4, dtype=torch.int64), torch.zeros(4)
    with pytest.raises(ValueError, match="kl_coef must be finite"):
        fused_linear_policy_loss(x, w, t, f, f, f, kl_coef=kl_coef)
