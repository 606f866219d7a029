"""Buffers that overlap: what a call refuses, and what it may be given in place."""
import ctypes

import numpy as np
import pytest

from test_gpu_kv4 import gpu, i32

pytestmark = pytest.mark.gpu

BAD = 6  # MRI_ERR_INVALID_ARGUMENT


def test_evict_refuses_overlapping_buffers(mri, gpu_ctx):
    import torch
    lib, h = gpu_ctx._lib, gpu_ctx.handle
    src, dst = mri.KVCache4(2, 2, 64, 256), mri.KVCache4(2, 2, 64, 64)
    lens, new = i32([256, 100, 0]), i32([0, 0, 0])
    kept = torch.zeros(2 * 2 * 64 + 2, dtype=torch.int32, device="cuda")

    def call(lens_at=None, new_at=None, kept_at=None, **of_dst):
        d = type(dst._desc)()
        ctypes.pointer(d)[0] = dst._desc
        for name, at in of_dst.items():
            setattr(d, name, at)
        return lib.mri_kv4_evict(h, src._ref, lens_at or lens.data_ptr(), ctypes.byref(d), 64, 8, new_at or new.data_ptr(),
                                 kept_at)

    torch.cuda.synchronize()
    launches = gpu_ctx.launch_count
    assert call(new_at=lens.data_ptr()) == BAD       # lengths in place
    assert call(new_at=lens.data_ptr() + 4) == BAD   # the second length is the first new one
    assert call(kept_at=lens.data_ptr()) == BAD
    assert call(new_at=kept.data_ptr() + 4 * 255, kept_at=kept.data_ptr()) == BAD
    for name in ("k", "v", "k_scale", "v_scale", "weight"):
        last = getattr(src, name)[-1, -1, -1].data_ptr() // 16 * 16
        assert call(**{name: last}) == BAD, name         # the source's last row
        assert call(**{name: src.weight.data_ptr()}) == BAD, name
    assert call(k=dst.v.data_ptr()) == BAD
    assert gpu_ctx.launch_count == launches
    # Side by side they are fine.
    assert call(new_at=kept.data_ptr() + 4 * 256, kept_at=kept.data_ptr()) == 0
    both = i32([200, 100, 0, 0])
    assert call(lens_at=both.data_ptr(), new_at=both.data_ptr() + 8) == 0
    gpu_ctx.synchronize()
    assert both.tolist() == [200, 100, 64, 64] and kept[-2:].tolist() == [64, 64]


def test_evict_into_a_part_of_the_same_buffers(mri, gpu_ctx):
    """Caches on entries of shared tensors: overlapping entries are refused, others move."""
    import torch
    big = mri.KVCache4(4, 2, 32, 128)
    big.weight.copy_(gpu(np.random.default_rng(0).random((4, 2, 128)).astype(np.float32)))
    part = lambda a, b: mri.KVCache4.from_tensors(*(t[a:b] for t in (big.k, big.v, big.k_scale, big.v_scale, big.weight)))  # noqa: E731
    with pytest.raises(ValueError):
        part(0, 2).evict(i32([128, 128]), part(1, 3), 16, 4)
    plain = mri.KVCache4(2, 2, 32, 128)
    _, want = part(0, 2).evict(i32([128, 90]), plain, 16, 4)
    _, kept = part(0, 2).evict(i32([128, 90]), part(2, 4), 16, 4)
    assert torch.equal(kept, want) and torch.equal(big.weight[2:, :, :16], plain.weight[:, :, :16])
