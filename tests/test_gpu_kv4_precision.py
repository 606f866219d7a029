"""Attention over the 4-bit cache where a bound relative to the largest value of
all would see nothing: blocks of 32 columns that are quieter than others, keys
that are quieter than others, and long runs of keys in one warp.

Bounds, fixed from the arithmetic before the first run, in units of 2^-23 (one
truncated float32 sum).  Scores: 24 A with A = scale * sum |q k|, as for all of
this attention's tests.  Weighted sums: the tensor core adds 16 keys a step, high
and low parts apart or one after the other, so n keys of one warp are at most n / 8
dependent sums; 32 more for P's exponential and its two halves, the row's
rescalings, the sums of partial results and the division.
"""
import numpy as np
import pytest

from test_gpu_kv4 import codec, gpu, i32

pytestmark = pytest.mark.gpu


def reference(q, k, v, n, scale):
    """One entry in float64: q [t, h, d], k and v [rows, kv, d].  out [t, h, d], the
    scores' A [t, h], and each row's softmax weights as a list [t][h]."""
    t, h, d = q.shape
    group = h // k.shape[1]
    out, a, weights = np.zeros(q.shape), np.zeros((t, h)), []
    for ti in range(t):
        seen, row = n - t + 1 + ti, []
        for hi in range(h):
            kk, vv = (x[:seen, hi // group].astype(np.float64) for x in (k, v))
            qq = q[ti, hi].astype(np.float64)
            z = kk @ qq * scale
            p = np.exp(z - z.max())
            p /= p.sum()
            out[ti, hi] = p @ vv
            a[ti, hi] = (np.abs(kk) @ np.abs(qq)).max() * abs(scale)
            row.append(p)
        weights.append(row)
    return out, a, weights


def cached(mri, k, v):
    """A cache of one entry with the rows k, v [rows, kv, d], and what it keeps of them."""
    cache = mri.KVCache4(1, k.shape[1], k.shape[2], k.shape[0])
    cache.append(gpu(k[None]), gpu(v[None]), i32([0]))
    return cache, codec(mri, k), codec(mri, v)


@pytest.mark.parametrize("tokens,heads", [(1, 4), (5, 4), (9, 8)])
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("apart", [9, 13, 18, 23])
def test_quiet_value_blocks(mri, gpu_ctx, tokens, heads, d, apart):
    """Blocks of 32 columns 2^apart below the loudest one, each as exact as its own values."""
    rng = np.random.default_rng(apart + d + tokens)
    n = 320
    k = rng.normal(0, 1, (n, 2, d)).astype(np.float32)
    quiet = np.exp2(-apart * np.arange(d // 32) / (d // 32 - 1))
    v = (rng.normal(0, 1, (n, 2, d)) * 2.0 ** 12 * np.repeat(quiet, 32)).astype(np.float32)
    q = rng.normal(0, 2, (tokens, heads, d)).astype(np.float32)
    cache, kk, vv = cached(mri, k, v)
    got = cache.attention(gpu(q[None]), i32([n])).cpu().numpy()[0]
    want, a, _ = reference(q, kk, vv, n, d ** -0.5)
    for b in range(d // 32):
        cols = slice(32 * b, 32 * b + 32)
        top = np.abs(vv[..., cols]).max()
        err = np.abs(got[..., cols] - want[..., cols]).max(-1)
        bound = (24 * a + n / 8 + 32) * 2.0 ** -23 * top
        assert (err <= bound).all(), f"block {b}: {(err / top).max():.3g} of its largest value, bound {(bound / top).min():.3g}"


@pytest.mark.parametrize("tokens", [1, 5])
@pytest.mark.parametrize("apart", [6, 10, 13])
def test_quiet_keys_beside_a_loud_one(mri, gpu_ctx, tokens, apart):
    """One key's values 2^apart above the others', with a weight below 2^-60.  P times a scale
    is held to 2^-25 where the row's largest P times the block's loudest scale is 2^9 at
    least: 2^(apart - 34) a key, of roundings that are independent of one another; n / 8 of
    them are more than twice the root of their sum of squares."""
    rng = np.random.default_rng(apart + tokens)
    n, d, heads = 320, 128, 4
    k = rng.normal(0, 1, (n, 1, d)).astype(np.float32)
    k[100] = -8.0
    v = rng.normal(0, 1, (n, 1, d)).astype(np.float32)
    v[100] *= 2.0 ** apart
    q = (rng.normal(0, 0.3, (tokens, heads, d)) + 1).astype(np.float32)
    cache, kk, vv = cached(mri, k, v)
    got = cache.attention(gpu(q[None]), i32([n])).cpu().numpy()[0]
    want, a, weights = reference(q, kk, vv, n, d ** -0.5)
    assert max(p[100] for row in weights for p in row) < 2.0 ** -60
    top = np.abs(np.delete(vv, 100, 0)).max()
    loudest = np.abs(vv[100]).max() / top
    err = np.abs(got - want).max(-1)
    bound = ((24 * a + n / 8 + 32) * 2.0 ** -23 + n * loudest * 2.0 ** -37) * top
    assert (err <= bound).all(), f"{(err / top).max():.3g} of the others' largest value, bound {(bound / top).min():.3g}"


@pytest.mark.parametrize("group", [2, 4])
def test_infinite_value_scale_that_rows_do_not_see(mri, gpu_ctx, group):
    """An infinite scale spoils its own block in the rows that see its key, and costs the
    others nothing: not a bit of theirs, one for one with the same call without it."""
    rng = np.random.default_rng(group)
    n, d, tokens = 320, 128, 4
    k, v = (rng.normal(0, 1, (n, 1, d)).astype(np.float32) for _ in range(2))
    q = rng.normal(0, 2, (tokens, group, d)).astype(np.float32)
    cache, kk, vv = cached(mri, k, v)
    clean = cache.attention(gpu(q[None]), i32([n])).cpu().numpy()[0]
    cache.v_scale[0, 0, n - 2, 1] = float("inf")  # seen by the last two tokens
    got = cache.attention(gpu(q[None]), i32([n])).cpu().numpy()[0]
    hit = np.zeros(got.shape, bool)
    hit[2:, :, 32:64] = True
    assert not np.isfinite(got[hit]).any()
    assert np.array_equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("tokens,group", [(1, 2), (5, 2)])
def test_sums_over_many_keys_of_a_warp(mri, gpu_ctx, tokens, group):
    """So many keys that a warp walks some 19000 of one head.  Sums that the tensor core cuts
    off drift by half a unit a step, 1200 steps of 16 keys; added to rounded ones every 512
    keys (8 rows: high and low parts have sums of their own) or 256 (16 rows: both in one)
    they are 32 cuts from that.  Without it both are off by more than the bound."""
    import torch
    heads, d, cap = 128, 128, 262144
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    cache = mri.KVCache4(1, heads, d, cap)
    # Value codes 8 to 15: values of one sign, so that a drift shows whole.
    cache.k.random_(0, 256, generator=gen)
    cache.v.random_(0, 256, generator=gen).bitwise_or_(0x88)
    cache.k_scale.fill_(0.25)
    cache.v_scale.copy_(torch.rand(cache.v_scale.shape, generator=gen, device="cuda") * 0.1 + 0.2)
    q = torch.randn(1, tokens, heads * group, d, generator=gen, device="cuda") * 0.02
    got = cache.attention(q, i32([cap]))
    for head in (0, 61, 127):
        one = mri.KVCache4.from_tensors(*(t[:, head:head + 1].contiguous() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale, cache.weight)))
        k, v = (t[0, :, 0].double() for t in one.read(None, cap))
        for t in range(tokens):
            seen = cap - tokens + 1 + t
            for g in range(group):
                row = q[0, t, head * group + g].double()
                a = float((k[:seen].abs() @ row.abs()).max()) * d ** -0.5
                want = torch.softmax(k[:seen] @ row * d ** -0.5, 0) @ v[:seen]
                err = ((got[0, t, head * group + g].double() - want).abs() / want).max()
                assert float(err) <= (24 * a + 32 + 32) * 2.0 ** -23, (head, t, g, float(err), a)
