"""The operators over a paged cache and packed prompts on the CPU, at the
ends of what they take."""
import pytest
import torch

import paged_limits as limits
import paged_oracle as oracle
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


@pytest.mark.parametrize("name", limits.DECODE_WILD)
def test_decode_wild_values(name):
    q, st, kw, want = limits.decode_wild(name)
    out = ops.paged_decode_op(q, st["k"], st["v"], st["table"], st["lens"],
                              **kw)
    oracle.check("out", out[0] if "mass" in kw else out, want["out"])


@pytest.mark.parametrize("name", limits.PACKED_WILD)
def test_packed_wild_values(name):
    args, kw, want = limits.packed_wild(name)
    oracle.check("out", ops.flash_prefill_packed_op(*args, **kw),
                 want["out"])
