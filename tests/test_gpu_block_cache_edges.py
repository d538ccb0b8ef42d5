"""Block-scaled cache operators where their arithmetic, argument or layout handling ends.

The helpers and their tolerances are those of test_gpu_block_cache.py.
"""

import pytest
import torch

from test_gpu_alibi import _kernel_names
from test_gpu_block_cache import run_attention

pytestmark = pytest.mark.gpu


def run_prefill(*args, **kw):
    """run_attention on a call that takes the 16-bit copy and the tcgen05 prefill."""
    got = []
    names = _kernel_names(lambda: got.append(run_attention(*args, **kw)))
    assert not names or any("block_copy_kernel" in n for n in names), names
    return got[0]


def dominant_key(nats, v_code, vs_exp=4):
    """Key 2 stands `nats` above all others; its V row holds one code throughout (0: it adds nothing to an output).

    The rest of an output row are the other keys' small probabilities, and the bound
    (relative to sum p |v| / sum p) asks for their own precision.
    """
    def mutate(q, kc, vc, ks, vs, table):
        page = table[0, 0].long()
        q[:, :, 0] = nats / (448 * 2.0 ** -7 * q.shape[-1] ** -0.5)
        raw = kc.view(torch.uint8)
        raw[..., 0] = 0
        raw[page, 2] = 0
        raw[page, 2, :, 0] = 0x7e                        # 448
        ks[page, 0] = 2.0 ** -7
        vc.view(torch.uint8)[page, 2] = v_code
        vs.fill_(2.0 ** vs_exp)                          # outputs stay normal numbers in f16
    return mutate


@pytest.mark.parametrize("v_code", [0, 1])
@pytest.mark.parametrize("nats", [4, 9, 12, 14, 16])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_dominant_key_without_value(dtype, nats, v_code):
    mutate = dominant_key(nats, v_code)
    for hq in (4, 8, 16, 24, 32):                        # every width of the decode kernel
        run_attention([1], [100], hq, 1, 128, 16, 16, dtype, mutate=mutate, q_scale=0.2)
    run_attention([3], [111], 4, 1, 256, 32, 32, dtype, mutate=mutate, q_scale=0.2)
    run_attention([2], [1900], 4, 2, 64, 16, 16, dtype, mutate=mutate, q_scale=0.2, window=100, first=4)
    run_attention([2], [1900], 4, 2, 128, 16, 16, dtype, mutate=mutate, q_scale=0.2, splits=3)


@pytest.mark.parametrize("nats", [4, 9, 12, 14])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_dominant_key_without_value_in_prompt_chunks(d, dtype, nats):
    mutate = dominant_key(nats, 0)
    run_prefill([130, 260], [170, 300], 32, 2, d, 16, 16, dtype, mutate=mutate, q_scale=0.2)
    run_prefill([130, 260], [500, 300], 32, 2, d, 16, 16, dtype, mutate=mutate, q_scale=0.2, window=90, first=4, sinks=True)
