"""The operators for batches beside an engine in one process."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_engine_leaves_the_errors_of_the_batch_operators(cuda, gpt2b):
    """A slot outside the paged cache is the serving program's error: an engine's run neither fails for it nor clears it."""
    from cuda_gpt2_inference_b200 import ops, weights
    from cuda_gpt2_inference_b200.engine import Engine
    cfg = weights.mini_config(L=2, NH=2, maxT=64, V=500, Vp=512)
    eng = Engine.from_buffer(weights.image(weights.synth_params(cfg, 3, init="test"), cfg, "bf16"), "bf16")
    want, _ = eng.generate([3, 141, 59], 8)
    assert gpt2b.device_error() == 0
    codes = torch.zeros(2, 2, 2, 16, 32, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(2, 2, 2, 16, 1, 2, dtype=torch.bfloat16, device="cuda")
    qkv = torch.zeros(1, 6 * 64, dtype=torch.bfloat16, device="cuda")
    ops.kv_cache_write_w4(codes, scales, qkv, torch.tensor([32], device="cuda"), 2)
    torch.cuda.synchronize()
    got, _ = eng.generate([3, 141, 59], 8)
    assert list(got) == list(want)
    assert gpt2b.device_error() == gpt2b.DEVERR_BAD_BLOCK
    assert gpt2b.device_error() == 0
    eng.close()
