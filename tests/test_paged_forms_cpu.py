"""Every form of attention over packed prompts and pages on the CPU."""
import pytest

import paged_forms as forms
import paged_oracle as oracle
from triton_dist_amd import ops


@pytest.mark.parametrize("name", forms.PACKED)
def test_packed(name):
    args, kw, want = forms.packed(name)
    got = ops.flash_prefill_packed_op(*args, return_lse=True, **kw)
    for x, key in zip(got, ("out", "lse")):
        oracle.check(key, x, want[key])


@pytest.mark.parametrize("name", forms.DECODE)
def test_decode(name):
    q, st, kw, want = forms.decode(name)
    got = ops.paged_decode_op(q, st["k"], st["v"], st["table"], st["lens"],
                              return_lse=True, **kw)
    for x, key in zip(got, ("out", "lse", "mass")):
        oracle.check(key, x, want[key])
