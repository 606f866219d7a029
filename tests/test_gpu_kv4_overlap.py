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


@pytest.mark.parametrize("tokens,heads,lens", [(1, 4, [1000, 3]), (7, 8, [1024, 900]), (70, 2, [512, 40])])
def test_attention_in_place_of_its_queries(mri, gpu_ctx, tokens, heads, lens):
    """out_dev == q_dev: right where nothing is tracked, refused where the queries are read again."""
    import torch
    rng = np.random.default_rng(tokens)
    cache = mri.KVCache4(2, 2, 64, 1024)
    x = gpu(rng.normal(0, 1, (2, 1024, 2, 64)).astype(np.float32))
    cache.append(x, x, i32([0, 0]))
    q, n, ld = gpu(rng.normal(0, 2, (2, tokens, heads, 64)).astype(np.float32)), i32(lens), heads * 64
    want = cache.attention(q, n)
    lib, h, ref = gpu_ctx._lib, gpu_ctx.handle, cache._ref
    torch.cuda.synchronize()
    launches = gpu_ctx.launch_count
    assert lib.mri_kv4_attention(h, ref, q.data_ptr(), ld, tokens, heads, n.data_ptr(), 0.125, 1, q.data_ptr()) == BAD
    assert gpu_ctx.launch_count == launches
    assert lib.mri_kv4_attention(h, ref, q.data_ptr(), ld, tokens, heads, n.data_ptr(), 0.125, 0, q.data_ptr()) == 0
    gpu_ctx.synchronize()
    assert torch.equal(q, want)


def test_attention_refuses_overlapping_buffers(mri, gpu_ctx):
    import torch
    cache = mri.KVCache4(2, 2, 64, 128)
    lib, h, ref = gpu_ctx._lib, gpu_ctx.handle, cache._ref
    n = i32([100, 128])
    rows = torch.zeros(8, 1024, device="cuda")  # queries in the first 256 of six rows
    q, spare = rows.data_ptr(), torch.zeros(2 * 3 * 256, device="cuda").data_ptr()

    def call(out, track=0, q_at=q, ld=1024, lens=None):
        return lib.mri_kv4_attention(h, ref, q_at, ld, 3, 4, lens or n.data_ptr(), 0.125, track, out)

    torch.cuda.synchronize()
    launches = gpu_ctx.launch_count
    row = 4 * 1024
    for out in (q, q + 4 * 255, q + row, q + 5 * row + 4 * 255, q - 4 * (2 * 3 * 256 - 1), cache.k.data_ptr(), cache.v.data_ptr() + 16,
                cache.weight.data_ptr(), n.data_ptr()):
        for track in (0, 1):
            assert call(out, track) == BAD, out - q
    assert call(spare, 1, q_at=cache.weight.data_ptr(), ld=256) == BAD  # queries in the totals
    assert call(spare, 1, lens=cache.weight.data_ptr()) == BAD
    assert gpu_ctx.launch_count == launches
    # Directly behind the last row's queries.
    assert call(q + 5 * row + 4 * 256) == 0
    assert call(spare) == 0
    gpu_ctx.synchronize()
