"""KV cache in 8 bits, beside test_gpu_cache8.py: many pieces of one sequence."""
import pytest
import torch

from test_gpu_cache8 import BF16, E4M3, F16, INT8, run_attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("old", [74000, 131040])
@pytest.mark.parametrize("dim,dtype,code", [(64, F16, E4M3), (128, BF16, INT8)])
def test_chunk_of_one_unit_behind_a_long_context(dim, dtype, code, old):
    """One KV head, one pair of query tiles: more pieces asked for than a merge has room for.  The call after it is not refused."""
    from flash_attn_triton_b200 import _native as N
    run_attend(11, [old], 32, True, 8, 1, dim, 256, 1, dtype, code, causal=True)
    torch.cuda.synchronize()
    assert N.lib().fa_device_wait_status(torch.cuda.current_device()) == 0
    run_attend(12, [100], 32, True, 8, 1, dim, 256, 1, dtype, code, causal=True)
