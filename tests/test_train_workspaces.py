"""Workspace sizes from Python (CPU only): what the library refuses raises, with its own words."""

import pytest

from purin_amd import _lib
from purin_amd.gradients import clip_workspace_bytes
from purin_amd.routing import route_workspace_bytes


def test_sizes_that_are_refused_raise():
    assert clip_workspace_bytes(0) > 0 and clip_workspace_bytes(500) > clip_workspace_bytes(1)
    with pytest.raises(_lib.PurinError, match="experts"):
        route_workspace_bytes(4, 0, 2)
    with pytest.raises(_lib.PurinError, match="tensors"):
        clip_workspace_bytes(-1)
