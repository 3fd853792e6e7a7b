"""Edges of the calls for many sequences (4-bit pages, packed prompts) on the GPU: what they refuse, and what they give
for tokens that they leave out."""
import random

import pytest
import torch

from innerq_amd import ops, paged
from oracle import serving_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float16, torch.bfloat16]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def randn(g, *shape, dtype=torch.float16):
    return torch.randn(*shape, generator=g).to(dtype).to(DEV)


@pytest.fixture(params=["native", "general"])
def front(request, monkeypatch):
    """The same calls through csrc/iq_pyfast.cpp and through the Python path alone."""
    if request.param == "general":
        monkeypatch.setattr(ops, "_native", lambda t: None)


@pytest.mark.parametrize("shape", [(0, 32), (10, 0), (0, 0)])
def test_empty_rotation_tables_are_refused(front, shape):
    """They are no "no rotation": nothing is appended."""
    g = torch.Generator().manual_seed(0)
    st = paged.PagedStore(2, 2, 64, DEV)
    st.pages.fill_(0x11111111)
    before = st.pages.clone()
    k, q = randn(g, 2, 2, 64), randn(g, 2, 4, 64)
    empty = torch.zeros(*shape, device=DEV)
    with pytest.raises(ValueError, match="rotation"):
        st.append(k, k, i32([[0], [1]]), i32([3, 4]), cos=empty, sin=empty, q=q)
    assert torch.equal(st.pages, before)
