"""The operators over a paged cache and packed prompts on the GPU, at the
ends of what they take."""
import pytest
import torch

import paged_limits as limits
from triton_dist_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", limits.LARGE)
def test_packed_large_logits(name):
    """Logits that 32 bits hold to many units: the largest takes it all, and
    equal ones share it."""
    args, kw, want = limits.packed_large(name)
    args = [x.cuda() for x in args]
    kw = {k: x.cuda() if isinstance(x, torch.Tensor) else x
          for k, x in kw.items()}
    out, lse = ops.flash_prefill_packed_op(*args, return_lse=True, **kw)
    limits.hold(out, lse, want)


@pytest.mark.parametrize("name", limits.LARGE)
def test_decode_large_logits(name):
    """The same, with equal keys in chunks apart, and their weights."""
    args, kw, want = limits.decode_large(name)
    args = [x.cuda() for x in args]
    kw = {k: x.cuda() if isinstance(x, torch.Tensor) else x
          for k, x in kw.items()}
    out, lse, mass = ops.paged_decode_op(*args, return_lse=True, **kw)
    limits.hold(out, lse, want)
    limits.hold_mass(mass, want)
