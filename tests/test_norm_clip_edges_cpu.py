"""The host side of hipops.group_norm, grad_norm and clip_grads at calls off the ordinary path."""
import pytest
import torch

import msnets_amd  # noqa: F401
from msnets_amd import hipops


def test_graphs_are_refused_in_grad_mode_only():
    p = torch.ones(3, requires_grad=True)
    with pytest.raises(ValueError, match="grads\\[2\\] requires a gradient"):
        hipops._refuse_graph(p * 2, "grads[2]")
    hipops._refuse_graph(p.detach(), "t")
    with torch.no_grad():
        hipops._refuse_graph(p, "t")
