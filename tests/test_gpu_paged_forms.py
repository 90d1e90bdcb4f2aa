"""Every form that the kernels of attention over packed prompts and pages are
built in, on the GPU."""
import pytest
import torch

import paged_forms as forms
import paged_oracle as oracle
from triton_dist_amd import ops

pytestmark = pytest.mark.gpu


def _cuda(x):
    return {k: _cuda(v) for k, v in x.items()} if isinstance(x, dict) else \
        x.cuda() if isinstance(x, torch.Tensor) else x


@pytest.mark.parametrize("name", forms.PACKED)
def test_packed(name):
    args, kw, want = forms.packed(name)
    got = ops.flash_prefill_packed_op(*(x.cuda() for x in args),
                                      return_lse=True, **_cuda(kw))
    for x, key in zip(got, ("out", "lse")):
        oracle.check(key, x, want[key])


@pytest.mark.parametrize("name", forms.DECODE)
def test_decode(name):
    q, st, kw, want = forms.decode(name)
    g = _cuda(st)
    got = ops.paged_decode_op(q.cuda(), g["k"], g["v"], g["table"],
                              g["lens"], return_lse=True, **_cuda(kw))
    for x, key in zip(got, ("out", "lse", "mass")):
        oracle.check(key, x, want[key])
