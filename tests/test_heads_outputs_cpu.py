"""Outputs of the caller of the norm and rotation of queries and keys: what is refused, without a GPU."""

from __future__ import annotations

import pytest
import torch

from foldforge_b200 import _lib, kernels

needs_library = pytest.mark.skipif(not (_lib.LIBRARY.exists() and (_lib.LIBRARY.parent / "_binding.so").exists()),
                                   reason="library not built")


# --------------------------------------------------------------------------- outputs that autograd follows
@needs_library
@pytest.mark.parametrize("leaf", [True, False])
def test_outputs_that_require_a_gradient_are_refused(leaf):
    """The calls record nothing: written in place, such a tensor would keep the gradient of what it held before."""
    table = kernels.rotary_table(kernels.rotary_frequencies(16), device="cpu")
    positions = torch.zeros(5, 1, dtype=torch.int64)
    q, k = torch.randn(5, 4, 16), torch.randn(5, 2, 16)
    followed = torch.randn(5, 4, 16, requires_grad=True)
    followed = followed if leaf else followed * 2
    other = torch.randn(5, 2, 16, requires_grad=True)

    def calls(q_out, k_out):
        return [lambda: kernels.rotary(q, k, positions, table, out=(q_out, k_out)),
                lambda: kernels.qk_norm_rotary(q, k, positions, table, None, None, out=(q_out, k_out)),
                lambda: kernels.qk_norm_rotary_backward(q, k, q, k, positions, table, None, None, out=(q_out, k_out))]

    for out in ((followed, None), (followed[:, :, :], torch.empty_like(k)), (None, other)):
        for call in calls(*out):
            with pytest.raises(_lib.UnsupportedCall, match="requires a gradient"):
                call()
        with torch.no_grad():  # nothing is recorded: only the device is missing here
            for call in calls(*out):
                with pytest.raises(_lib.UnsupportedCall, match="CUDA device"):
                    call()
