"""Calls of the operators for batches that would overwrite what they read, or that the header does not allow (no GPU:
refused before any launch)."""
from __future__ import annotations

import pytest

FAR = 1 << 40


def _addresses(names):
    return {n: (i + 1) * FAR for i, n in enumerate(names)}  # far apart, 16-byte aligned, never read


def _clash(call, at, ok, writes, reads, refused):
    """Every output on every input and on every other output, as a whole and by a byte."""
    for w in writes:
        for r in [*reads, *[x for x in writes if x != w]]:
            for by in (0, 16):
                assert call({**at, w: at[r] + by}) == refused, (w, r, by)
    assert call(at) != refused and ok(call(at))


def _not_refused(gpt2b):
    # without a GPU the launch fails, with one nothing may be launched on these addresses: only the CPU run calls it
    return lambda rc: rc >= gpt2b.ERR_CUDA


@pytest.fixture()
def no_gpu():
    import torch
    if torch.cuda.is_available():
        pytest.skip("calls with made-up addresses that pass the checks")


def test_verify_outputs_over_inputs(gpt2b, no_gpu):
    names = ["out", "n", "tokens", "p", "q", "start", "ua", "us"]

    def call(a):
        return gpt2b.lib().gpt2b_verify_draft_tokens(*[a[n] for n in names], 8, 16, 100, 128, 128, 6, None)

    _clash(call, _addresses(names), _not_refused(gpt2b), ["out", "n"], names[2:], gpt2b.ERR_INVALID_ARG)


def test_table_outputs_over_each_other(gpt2b, no_gpu):
    names = ["table", "slots", "positions", "start", "lens", "blocks", "left", "ctx", "new", "have", "free", "count"]

    def call(a):
        return gpt2b.lib().gpt2b_kv_block_tables(*[a[n] for n in names], 8, 16, 16, 100, 64, None)

    # by a byte range: `left` and `count` are 4 bytes, so only the same address clashes with them
    at = _addresses(names)
    for w in names[:7]:
        for r in names:
            if r != w:
                assert call({**at, w: at[r]}) == gpt2b.ERR_INVALID_ARG, (w, r)
    assert _not_refused(gpt2b)(call(at))


@pytest.mark.parametrize("rows", [1, 100])
def test_cache_and_attention_outputs_over_inputs(gpt2b, no_gpu, rows):
    lib = gpt2b.lib()

    def write(a):
        return lib.gpt2b_kv_cache_write_w4(a["codes"], a["scales"], a["qkv"], a["slots"], rows, 4, 2, 64, 512, 8, 16, None)

    def read(a):
        return lib.gpt2b_kv_cache_read_w4(a["out"], a["codes"], a["scales"], a["slots"], rows, 2, 64, 8, 16, None)

    def attend(a):
        return lib.gpt2b_attention_forward_paged_w4(a["out"], a["qkv"], a["codes"], a["scales"], a["table"], a["lens"], a["start"],
                                                    8, rows, 4, 2, 64, 512, 8, 16, 16, 4, 0.125, a["ws"], 1 << 30, None)

    at = _addresses(["out", "codes", "scales", "qkv", "slots", "table", "lens", "start", "ws"])
    bad, ok = gpt2b.ERR_INVALID_ARG, _not_refused(gpt2b)
    slots = ["slots"] if rows > 2 else []  # (8 bytes: the byte further clashes with nothing)
    _clash(write, at, ok, ["codes", "scales"], ["qkv", *slots], bad)
    _clash(read, at, ok, ["out"], ["codes", "scales", *slots], bad)
    _clash(attend, at, ok, ["out", "ws"], ["qkv", "codes", "scales", "table", "lens", "start"], bad)
    # an empty step touches nothing
    assert lib.gpt2b_kv_cache_write_w4(FAR, FAR, FAR, FAR, 0, 4, 2, 64, 512, 8, 16, None) == gpt2b.OK


def test_temperature_that_32_bits_hold_as_zero(gpt2b):
    """0 asks for the largest logit; a positive temperature below FP32's range is refused, not taken for it."""
    import torch

    from cuda_gpt2_inference_b200 import ops
    x = torch.zeros(2, 9)
    for T in (1e-46, 1e-300, -1e-60):
        with pytest.raises(gpt2b.Gpt2bError, match="temperature") as e:
            ops.softmax_probs(x, x.clone(), T)
        assert e.value.status == gpt2b.ERR_INVALID_ARG
    with pytest.raises(gpt2b.Gpt2bError, match="CUDA"):  # what is allowed comes as far as the tensors' device
        ops.softmax_probs(x, x.clone(), 0.0)
