"""What log probabilities refuse before any look at a device."""
import pytest
import torch

from turbovec_amd import _lib as T
from turbovec_amd import sampling


@pytest.mark.parametrize("which", ["scores", "temperature"])
def test_forward_mode_is_refused(which):
    """A tangent that is dropped would read as zero; outside of its level a tensor has none."""
    from torch.autograd import forward_ad
    x, t, slots = torch.zeros(3, 256), torch.ones(3), torch.zeros(3, dtype=torch.int64)
    for leaf in (False, True):
        with forward_ad.dual_level():
            scores, temperature = x.clone().requires_grad_(leaf), t.clone()
            if which == "scores":
                scores = forward_ad.make_dual(scores, torch.ones_like(x))
            else:
                temperature = forward_ad.make_dual(temperature, torch.ones_like(t))
            with pytest.raises(ValueError, match=f"{which}: log_probs has no forward-mode"):
                sampling.log_probs(scores, slots, temperature=temperature)
            with pytest.raises(ValueError, match="on a GPU"):
                sampling.log_probs(x, slots, temperature=t)


@pytest.mark.parametrize("rows,n,top,parts", [(1, 32_000, 0, False), (1, 100_000, 0, True), (1, 100_000, 20, False), (1, 128_256, 20, True), (64, 128_256, 0, True), (64, 128_256, 20, False),
                                              (200, 1_000_000, 0, False), (1, 1_000_000, 128, True), (1, 8192, 20, False)])
def test_rows_in_parts_go_by_what_is_asked_for(rows, n, top, parts):
    """A call needs a workspace where rows are read in parts: from fewer scores on without alternatives, whose ranking parts do twice."""
    need = T.lib().tv_log_probs_workspace(rows, n, top)
    assert (need > 0) == parts
    assert need % (rows * (16 + 8 * top)) == 0
