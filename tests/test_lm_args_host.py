"""Arguments of the layered decoders' calls (no GPU)."""
import numpy as np
import pytest
import torch


@pytest.mark.parametrize("scale", [np.float32(0.25), np.float64(0.25), torch.tensor(0.25), 1], ids=["float32", "float64", "tensor", "whole"])
def test_a_scale_of_any_number_type(scale):
    """The general kernel's and the rotated forms' arguments are made in Python."""
    from msa_b200 import lm_ops as K
    q, k, i = torch.zeros((3, 4, 8)), torch.zeros((3, 2, 8)), torch.zeros(4, dtype=torch.int32)
    for qb, kb in ((None, None), (q[:, :, :4], k[:, :1, :4])):
        a = K.attn_args(q, qb, k, kb, k, q, scale=scale, window=5, start=i, cu=i, seq0=0, seq1=1, max_len=3, ctx_off=i)
        assert a.scale == float(scale) and a.group == 2 and a.db == (4 if qb is not None else 0)
