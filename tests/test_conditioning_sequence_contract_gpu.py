"""What the sequence operators promise beside their values: state that belongs to others, streams that rest, calls at the edges of what is allowed."""
import ctypes
import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import sequence_reference as ref
from genefaceplusplus_amd import _lib
from genefaceplusplus_amd._lib import GfppError
from genefaceplusplus_amd.radnerfs import RotaryEncoder, WindowCache, layer_norm, window_attention, window_attention_step

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


# ---- sizes at the edges ----------------------------------------------------------------------------------------------------------------------------------------
def test_layer_norm_of_very_wide_rows():
    """More columns than 2^16 workgroups of the column sums take side by side, more than 2^32 threads of the last launch."""
    N = 2 ** 26 + 35
    x, w, b, dy = rand(0, 1, N), rand(1, N), rand(2, N), rand(3, 1, N)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(db, dy[0])
    want = ref.layer_norm(x.detach(), w.detach(), b.detach(), 1e-5, dy)
    for name, got in (("y", y), ("dx", dx), ("dweight", dw)):
        value, bound = want[name]
        assert ((got.detach().double() - value).abs() <= bound).all(), name
