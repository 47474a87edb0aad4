"""Gradients of gradients of the attention calls: there are none, and whoever asks is told."""
import random

import pytest
import torch

import flash_attn_triton_b200 as fa
from test_gpu_drafting_more import refuses_second_gradients
from util import DEV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("behind", [0, 1])                     # 1: not on a 16-byte boundary, so that the call works on copies
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("call", ["dense", "dropout", "qkv", "kv", "varlen"])
def test_gradients_of_gradients_of_attention_are_refused(call, dtype, behind):
    flat = torch.randn(70 * 3 * 2 * 64 + behind, generator=torch.Generator().manual_seed(4)).to(dtype).to(DEV)
    leaf = flat[behind:].view(1, 70, 3, 2, 64).requires_grad_()
    cu = torch.tensor([0, 30, 70], dtype=torch.int32, device=DEV)

    def dropped(x):
        random.seed(5)                                        # where a call draws its seed
        return fa.flash_attn_func(*x.unbind(2), dropout_p=0.2)
    calls = dict(dense=lambda x: fa.flash_attn_func(*x.unbind(2)), dropout=dropped, qkv=fa.flash_attn_qkvpacked_func,
                 kv=lambda x: fa.flash_attn_kvpacked_func(x[:, :, 0], x[:, :, 1:]),
                 varlen=lambda x: fa.flash_attn_varlen_func(*x[0].unbind(1), cu, cu, 40, 40))
    refuses_second_gradients(calls[call], leaf)
