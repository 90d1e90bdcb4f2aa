"""The operators over a paged cache and packed prompts on the CPU, at the
ends of what they take."""
import pytest
import torch

import paged_limits as limits
from triton_dist_amd import ops


@pytest.mark.parametrize("name", limits.LARGE)
def test_packed_large_logits(name):
    args, kw, want = limits.packed_large(name)
    out, lse = ops.flash_prefill_packed_op(*args, return_lse=True, **kw)
    limits.hold(out, lse, want)


@pytest.mark.parametrize("name", limits.LARGE)
def test_decode_large_logits(name):
    args, kw, want = limits.decode_large(name)
    out, lse, mass = ops.paged_decode_op(*args, return_lse=True, **kw)
    limits.hold(out, lse, want)
    limits.hold_mass(mass, want)
