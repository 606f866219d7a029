"""CUDA graphs that captured calls of a context whose scratch grows later."""
import numpy as np
import pytest

from test_gpu_kv4 import gpu, i32

pytestmark = pytest.mark.gpu


def cache_of(mri, rng, ctx, batch, heads, d, capacity, fill):
    cache = mri.KVCache4(batch, heads, d, capacity, ctx=ctx)
    x = [gpu(rng.normal(0, 1, (batch, fill, heads, d)).astype(np.float32)) for _ in range(2)]
    cache.append(*x, i32([0] * batch))
    return cache


@pytest.mark.parametrize("tokens", [1, 5])
def test_replay_after_the_scratch_has_grown(mri, gpu_ctx, tokens):
    """A step is captured; then a tracked prompt chunk that needs far more scratch runs on the
    same context, and memory of the old size is allocated and filled; the replay still
    gives what the step gives outside a graph."""
    import torch
    rng = np.random.default_rng(tokens)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ctx = mri.Context(0, stream=s)
        cache = cache_of(mri, rng, ctx, 2, 2, 64, 4096, 4000)
        big = cache_of(mri, rng, ctx, 2, 8, 128, 2048, 2048)
        small = mri.KVCache4(2, 2, 64, 256, ctx=ctx)
        q = gpu(rng.normal(0, 2, (2, tokens, 4, 64)).astype(np.float32))
        lens = i32([4000, 777])
        new_lens = torch.empty_like(lens)

        def step():
            out = cache.attention(q, lens, track=True)
            # With no place for the kept positions eviction holds them in scratch.
            mri._check(ctx._lib.mri_kv4_evict(ctx.handle, cache._ref, lens.data_ptr(), small._ref, 200, 16,
                                              new_lens.data_ptr(), None))
            return out

        cache.weight.zero_()
        want = step().clone()
        rows = [t.clone() for t in (small.k, small.v, small.weight)]
        cache.weight.zero_()
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = step()
        g.replay()
        s.synchronize()
        assert torch.equal(out, want)
        q_big, lens_big = gpu(rng.normal(0, 2, (2, 1024, 64, 128)).astype(np.float32)), i32([2048, 1500])
        room = torch.empty_like(q_big)  # torch keeps this memory for the output
        del room
        free = torch.cuda.mem_get_info()[0]
        big.attention(q_big, lens_big, track=True)
        s.synchronize()
        assert torch.cuda.mem_get_info()[0] < free - (64 << 20)  # it did grow
        filled = [torch.full((4 << 20,), float("nan"), device="cuda") for _ in range(32)]
        cache.weight.zero_()
        for t in (out, small.k, small.v, small.weight, new_lens):
            t.zero_()
        g.replay()
        s.synchronize()
        assert torch.equal(out, want) and new_lens.tolist() == [200, 200]
        assert all(torch.equal(a, b) for a, b in zip((small.k, small.v, small.weight), rows))
        assert all(bool(t.isnan().all()) for t in filled)
        # And the context's own calls go on as before, in the grown scratch.
        cache.weight.zero_()
        assert torch.equal(step(), want)
        s.synchronize()
        del g
    s.synchronize()


def test_capture_of_a_call_that_would_grow_the_scratch(mri, gpu_ctx):
    """It is refused; the capture itself and the context stay usable."""
    import torch
    rng = np.random.default_rng(0)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ctx = mri.Context(0, stream=s)
        cache = cache_of(mri, rng, ctx, 1, 2, 64, 256, 200)
        q = gpu(rng.normal(0, 2, (1, 1, 4, 64)).astype(np.float32))
        lens = i32([200])
        s.synchronize()
        g, x = torch.cuda.CUDAGraph(), torch.zeros(4, device="cuda")
        s.synchronize()
        with torch.cuda.graph(g, stream=s):
            with pytest.raises(mri.CudaError, match="before the capture"):
                cache.attention(q, lens)
            x.add_(1)
        g.replay()
        s.synchronize()
        assert x.tolist() == [1.0] * 4
        want = cache.attention(q, lens).clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = cache.attention(q, lens)
        g.replay()
        s.synchronize()
        assert torch.equal(out, want)
        del g
    s.synchronize()
