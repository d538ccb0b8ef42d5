"""Block-scaled cache operators on the CPU: host checks, the axis map, and the host oracle against itself."""

import ctypes
import weakref

import numpy as np
import pytest
import torch

from flash_attn_b200 import _capi
from flash_attn_b200 import (append_kvcache_block_scaled, flash_attn_with_block_scaled_kvcache, rotary_axis_map,
                             verify_draft_tokens)
from flash_attn_b200 import block_cache
from oracle import block_cache as ob


def test_struct_layouts_match_the_header():
    # fa_tensor is 80 bytes; scalars of 4 bytes, the struct 8-byte aligned.
    assert block_cache._APPEND.size == 15 * 80 + 16
    assert block_cache._ATTEND.size == 12 * 80 + 32
    assert block_cache._VERIFY.size == 10 * 80 + 8


def test_exchanged_descriptors_match_the_attributes():
    """fa_describe through torch's exchange function gives what reading a tensor's attributes gives."""
    exchange = _capi.exchange_function()
    if exchange is None:
        pytest.skip("this torch has no DLPack exchange function")
    base = torch.arange(2 * 6 * 8 * 10)
    tensors = [base.view(2, 6, 8, 10).to(dt) for dt in (torch.float32, torch.float16, torch.bfloat16, torch.int32,
                                                       torch.int64, torch.uint8)]
    tensors += [tensors[0].to(torch.float8_e4m3fn), tensors[0][:, 1::2, ::3], tensors[1].permute(3, 1, 0, 2)[2:5],
                tensors[3][1, 2], torch.zeros(0, 4), torch.zeros(5)[3:], torch.tensor(3.0), base > 3,
                tensors[2][:, :, :1].expand(2, 6, 8, 10)]
    objects = tensors + [None]
    out = (_capi.Tensor * len(objects))()
    describe = _capi.describe_function()
    describe.argtypes = [ctypes.c_void_p, ctypes.c_int32, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int32]
    ids = (ctypes.c_void_p * len(objects))(*[None if t is None else id(t) for t in objects])
    assert describe(ids, len(objects), exchange, out, 1) == 0
    for t, got in zip(objects, out):
        want = _capi.tensor(t)
        assert got.dtype == want.dtype and got.ndim == want.ndim
        assert list(got.shape) == list(want.shape)
        if t is not None and t.numel():
            assert got.ptr == want.ptr
            for n, a, b in zip(want.shape, got.stride, want.stride):
                assert a == b or n <= 1, (t.shape, t.stride(), list(got.stride))
    assert describe(ids, len(objects), exchange, out, 0) == _capi.FA_ERR_INVALID    # CPU tensors


def test_axis_map():
    assert rotary_axis_map([2, 1, 1]).tolist() == [0, 0, 1, 2]
    assert rotary_axis_map([3, 2, 1], interleaved=True).tolist() == [0, 1, 2, 0, 1, 0]
    assert rotary_axis_map([0, 2]).tolist() == [1, 1]
    with pytest.raises(ValueError):
        rotary_axis_map([])
    with pytest.raises(ValueError):
        rotary_axis_map([2, -1])


def test_cpu_tensors_and_gradients_are_refused():
    cache = torch.zeros(2, 16, 1, 64).to(torch.float8_e4m3fn)
    scale = torch.ones(2, 1, 1)
    q = torch.randn(1, 1, 2, 64)
    lens, table = torch.ones(1, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        flash_attn_with_block_scaled_kvcache(q, cache, cache, scale, scale, lens, table)
    with pytest.raises(ValueError, match="CUDA"):
        append_kvcache_block_scaled(q[:, :, :1], q[:, :, :1], cache, cache, scale, scale, lens, table)
    with pytest.raises(ValueError, match="CUDA"):
        verify_draft_tokens(torch.randn(1, 5), torch.zeros(0, dtype=torch.int32), torch.zeros(2, dtype=torch.int32),
                            torch.zeros(0), torch.ones(1, 5), max_draft=1)


def test_oracle_scale_is_the_least_power_of_two():
    for amax in (0.0, 1e-40, 1.0, 447.9, 448.0, 448.1, 896.0, 1e30, 3e38):
        s = ob.scale_of(amax)
        assert amax <= 448 * s or s == 2.0 ** 100
        assert s == 2.0 ** -100 or amax > 224 * s


def test_oracle_rescale_is_exact_for_normal_codes():
    """Doubling a block's scale keeps every code that stays normal."""
    g = np.random.default_rng(0)
    codes = [g.integers(24, 120, (1, 16, 1, 16)).astype(np.uint8) for _ in range(2)]
    scales = [np.full((1, 1, 1), 0.25, dtype=np.float32) for _ in range(2)]
    was = ob.e4m3_decode(codes[0][0, :3]) * 0.25
    x = np.full((1, 1, 16), 200.0, dtype=np.float32)
    ob.append(x, x, None, codes, scales, [3], np.zeros((1, 1), dtype=np.int32), [0, 1])
    assert scales[0][0, 0, 0] == 0.5
    assert np.array_equal(ob.e4m3_decode(codes[0][0, :3]) * 0.5, was)


def test_oracle_verification_samples_the_target():
    """Over many random numbers the first token follows the target's distribution, whatever the draft."""
    g = np.random.default_rng(1)
    V, n = 5, 4000
    logits = np.tile(np.array([[0.3, 1.2, -0.5, 0.0, 0.8]]), (2 * n, 1))
    q = np.tile(np.array([[0.5, 0.1, 0.2, 0.1, 0.1]]), (n, 1))
    tokens = np.array([g.choice(V, p=q[0]) for _ in range(n)])
    out, accepted, _ = ob.verify(logits, tokens, np.arange(n + 1), g.random(n), g.exponential(size=(n, V)), q, None, 1)
    p = np.exp(logits[0]) / np.exp(logits[0]).sum()
    got = np.bincount(out[:, 0], minlength=V) / n
    assert np.abs(got - p).max() < 5 * np.sqrt(0.25 / n)
    assert 0 < accepted.mean() < 1


def test_packed_copies_live_until_the_launch(monkeypatch):
    """Head-major keys, values and queries are copied into packed rows; the copies must not be freed before the launch."""
    made, alive = [], []
    packed = block_cache._packed

    def watched(x, name):
        out = packed(x, name)
        made.append(weakref.ref(out))
        return out

    def launch(fn, view, index):
        alive.extend(ref() is not None for ref in made)
    monkeypatch.setattr(block_cache, "_packed", watched)
    monkeypatch.setattr(block_cache, "_cuda_index", lambda x: 0)
    monkeypatch.setattr(block_cache, "_call", launch)
    monkeypatch.setattr(block_cache._Arguments, "pack", lambda self, tensors, scalars, index: (None, None))
    x = torch.randn(2, 3, 5, 64).transpose(1, 2)             # [batch, new, heads, dim], heads outermost in memory
    cache, scale = torch.zeros(2, 16, 3, 64).to(torch.float8_e4m3fn), torch.ones(2, 1, 3)
    append_kvcache_block_scaled(x, x, cache, cache, scale, scale, torch.zeros(2, dtype=torch.int32),
                                torch.zeros(2, 2, dtype=torch.int32), query=x)
    assert len(made) == 4 and all(alive) and len(alive) == 4


@pytest.mark.parametrize("scalars", [(1, 2 ** 31, 0), (1, 2.5, 0), (1, None, 0), (-2 ** 31 - 1, 1, 0)])
def test_numbers_that_do_not_fit_are_refused(scalars):
    with pytest.raises(ValueError, match="32-bit"):
        block_cache._APPEND.pack([None] * 15, scalars, 0)
