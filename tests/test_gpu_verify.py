"""Verification of drafted tokens on the GPU against the rule in numpy float64.

Tokens must be equal wherever the rule's decision has a margin: a uniform that
lies within 1e-5 of the acceptance probability, or two candidates within 1e-5
of each other, could go either way in float32, and the inputs of these tests
are checked to have none (else the seed is to be changed in the test, not the
tolerance).  logprobs: a float32 softmax over up to 1e5 values, within 1e-5 *
(1 + |logprob|).
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def gpu(a):
    import torch
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def rule(logits, drafts, uniforms, races, q, temp):
    """(tokens, accepted, logprobs, smallest margin) of one sequence."""
    k, vocab = drafts.size, logits.shape[1]
    x = logits.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, float(np.finfo(np.float32).max)))
    greedy = temp == 0
    t = temp if temp > 0 and np.isfinite(temp) else 1.0
    tokens, said, margin = np.full(k + 1, -1), np.zeros(k + 1), np.inf
    for j in range(k + 1):
        z = (x[j] - x[j].max()) / t
        logp = z - np.log(np.exp(z).sum())
        p = np.exp(logp)
        best = int(x[j].argmax())
        ok = False
        if j < k and 0 <= drafts[j] < vocab:
            d = int(drafts[j])
            if greedy:
                ok = d == best
            else:
                level = uniforms[j].astype(np.float64) * (1.0 if q is None else float(q[j, d]))
                ok = level < p[d]
                if max(level, p[d]) > 0:
                    margin = min(margin, abs(level - p[d]) / max(level, p[d]))
        if ok:
            tokens[j], said[j] = d, logp[d]
            continue
        w = p
        if j < k and not greedy:
            if q is not None:
                w = np.maximum(p - q[j].astype(np.float64), 0)
            elif 0 <= drafts[j] < vocab:
                w = p.copy()
                w[drafts[j]] = 0
            if not w.max() > 0:
                w = p
        if greedy:
            pick = best
        else:
            r = w / races.astype(np.float64)
            pick = int(r.argmax())
            rest = np.delete(r, pick)
            if rest.size and r[pick] > 0:
                margin = min(margin, (r[pick] - rest.max()) / r[pick])
        tokens[j], said[j] = pick, logp[pick]
        return tokens, j, said, margin
    raise AssertionError


def check(mri, logits, drafts, uniforms, races, q=None, temp=None, ctx=None):
    b = logits.shape[0]
    got = mri.verify_draft(gpu(logits), gpu(drafts), gpu(uniforms), gpu(races), draft_probs=gpu(q), temperature=gpu(temp),
                           ctx=ctx)
    tokens, accepted, logprobs = (t.cpu().numpy() for t in got)
    for i in range(b):
        want = rule(logits[i], drafts[i], uniforms[i], races[i], None if q is None else q[i], 1.0 if temp is None else temp[i])
        assert want[3] > 1e-5, f"entry {i}: margin {want[3]:.2g}; use another seed"
        assert tokens[i].tolist() == want[0].tolist(), i
        assert accepted[i] == want[1]
        assert (np.abs(logprobs[i] - want[2]) <= 1e-5 * (1 + np.abs(want[2]))).all()
    return accepted


def inputs(rng, b, k, vocab, sampled=True, spread=2.5, apart=0.5):
    base = rng.normal(0, spread, (b, k + 1, vocab))
    logits = (base + rng.normal(0, apart, base.shape)).astype(np.float32)
    draft = base[:, :k] + rng.normal(0, apart, (b, k, vocab))
    q = np.exp(draft - draft.max(-1, keepdims=True)) if k else np.zeros((b, 0, vocab))
    q = (q / q.sum(-1, keepdims=True)).astype(np.float32) if k else q.astype(np.float32)
    drafts = np.array([[rng.choice(vocab, p=q[i, j].astype(np.float64) / q[i, j].astype(np.float64).sum()) for j in range(k)]
                       for i in range(b)], np.int32).reshape(b, k)
    return logits, drafts, rng.random((b, k)).astype(np.float32), rng.exponential(1, (b, vocab)).astype(np.float32), \
        q if sampled else None


@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4097, 32000, 50001])
@pytest.mark.parametrize("b,k", [(1, 1), (3, 4), (9, 7)])
def test_sampled_drafts(mri, gpu_ctx, b, k, vocab):
    rng = np.random.default_rng(b * vocab + k)
    logits, drafts, u, e, q = inputs(rng, b, k, vocab)
    temp = rng.uniform(0.6, 1.2, b).astype(np.float32)
    check(mri, logits, drafts, u, e, q, temp)
    check(mri, logits, drafts, u, e, q, None)


@pytest.mark.parametrize("b,k,vocab", [(160, 1, 4100), (40, 1, 20001), (200, 1, 20004), (700, 1, 301), (2, 1, 140001), (2, 1, 131072)])
def test_batches_and_long_rows(mri, gpu_ctx, b, k, vocab):
    """Sequences split over 1 to 8 blocks, rows of one pass and of several."""
    rng = np.random.default_rng(b + vocab)
    logits, drafts, u, e, q = inputs(rng, b, k, vocab)
    temp = np.where(np.arange(b) % 5 == 4, 0.0, rng.uniform(0.6, 1.2, b)).astype(np.float32)
    logits[::3, :, ::7] = -np.inf
    logits[1::3, :, : vocab // 2] = np.nan
    q[::3, :, ::7] = 0
    check(mri, logits, drafts, u, e, q, temp)
    check(mri, logits, drafts, u, e, None, temp)


@pytest.mark.parametrize("vocab", [33, 32000])
def test_chosen_drafts_and_greedy_entries(mri, gpu_ctx, vocab):
    rng = np.random.default_rng(vocab)
    logits, drafts, u, e, _ = inputs(rng, 12, 3, vocab, sampled=False)
    best = logits[:, :3].argmax(-1).astype(np.int32)
    drafts = np.where(rng.random(drafts.shape) < 0.6, best, drafts).astype(np.int32)
    temp = np.where(np.arange(12) % 2 == 0, 0.0, 0.9).astype(np.float32)
    accepted = check(mri, logits, drafts, u, e, None, temp)
    assert accepted.max() > accepted.min()


def test_no_drafts(mri, gpu_ctx):
    """n_drafts = 0 samples one token from the target."""
    rng = np.random.default_rng(0)
    logits, drafts, u, e, q = inputs(rng, 4, 0, 777)
    check(mri, logits, drafts, u, e, None, np.array([0, 1, 0.5, 2], np.float32))


def test_all_accepted_and_none(mri, gpu_ctx):
    rng = np.random.default_rng(1)
    logits, drafts, u, e, q = inputs(rng, 6, 64, 257)
    assert (check(mri, logits, drafts, np.zeros_like(u), e, q) == 64).all()
    q[...] = 1.0  # p < u q wherever u is near 1
    assert (check(mri, logits, drafts, np.full_like(u, 0.9999), e, q) == 0).all()


def test_equal_distributions(mri, gpu_ctx):
    """The draft model is the target: with u below 1 every draft stands."""
    rng = np.random.default_rng(2)
    logits, drafts, u, e, _ = inputs(rng, 3, 4, 500)
    z = logits[:, :4] - logits[:, :4].max(-1, keepdims=True)
    q = np.exp(z) / np.exp(z).sum(-1, keepdims=True)
    assert (check(mri, logits, drafts, u * np.float32(0.99), e, q.astype(np.float32)) == 4).all()


def test_masked_logits(mri, gpu_ctx):
    """-inf, NaN and +inf logits: probability 0, probability 0, a share of all of it."""
    rng = np.random.default_rng(3)
    logits, drafts, u, e, _ = inputs(rng, 5, 2, 300, sampled=False)
    logits[0, :, 10:] = -np.inf
    logits[1, 0, ::2] = np.nan
    logits[2, :, 7] = np.inf
    logits[3, 1, :] = -np.inf
    logits[3, 1, 299] = -4.0
    logits[4, 0, drafts[4, 0]] = -np.inf
    drafts[2, 0] = 7
    check(mri, logits, drafts, u, e, None)


def test_ties_go_to_the_lowest_index(mri, gpu_ctx):
    vocab = 40000
    logits = np.zeros((2, 2, vocab), np.float32)
    logits[:, :, 5000] = logits[:, :, 12345] = logits[:, :, 39999] = 3.0
    races = np.ones((2, vocab), np.float32)
    drafts = np.array([[5000], [12345]], np.int32)
    for temp, want, accepted in ((0.0, [[5000, 5000], [5000, -1]], [1, 0]), (1.0, [[12345, -1], [5000, -1]], [0, 0])):
        t, n, _ = mri.verify_draft(gpu(logits), gpu(drafts), gpu(np.full((2, 1), 0.999, np.float32)), gpu(races),
                                   temperature=gpu(np.full(2, temp, np.float32)))
        assert n.cpu().tolist() == accepted
        assert t.cpu().tolist() == want


def test_drafts_outside_the_vocabulary(mri, gpu_ctx):
    rng = np.random.default_rng(5)
    logits, drafts, u, e, q = inputs(rng, 4, 2, 100)
    drafts[0, 0], drafts[1, 1], drafts[2, 0], drafts[3, 0] = -1, 100, 2 ** 31 - 1, -2 ** 31
    check(mri, logits, drafts, u, e, None)
    check(mri, logits, drafts, u, e, q)


def test_odd_temperatures(mri, gpu_ctx):
    """Negative and non-finite temperatures count as 1; tiny ones are near greedy."""
    rng = np.random.default_rng(6)
    logits, drafts, u, e, _ = inputs(rng, 5, 2, 100, sampled=False)
    check(mri, logits, drafts, u, e, None, np.array([-1, np.nan, np.inf, 1e-3, 50], np.float32))


def test_subnormal_temperatures(mri, gpu_ctx):
    """1 / t, or its product with log2 e, is past float32: the draws are those of the largest logits."""
    rng = np.random.default_rng(12)
    logits, drafts, u, e, _ = inputs(rng, 6, 2, 100, sampled=False)
    drafts[::2] = logits[::2, :2].argmax(-1)
    temp = np.array([4.1e-39, 2.9e-39, 1e-39, 1e-42, 1.4e-45, 1.2e-38], np.float32)
    accepted = check(mri, logits, drafts, u, e, None, temp)
    assert (accepted[::2] == 2).all()
    # Equal largest logits share the probability.
    logits[:, :, 17] = logits[:, :, 61] = 9.0
    accepted = check(mri, logits, np.full_like(drafts, 61), np.full_like(u, 0.49), e, None, temp)
    assert (accepted == 2).sum() >= 4
    t, n, lp = (x.cpu().numpy() for x in mri.verify_draft(gpu(logits), gpu(np.full_like(drafts, 61)), gpu(np.full_like(u, 0.49)),
                                                          gpu(e), temperature=gpu(temp)))
    for i in np.flatnonzero(logits.max((1, 2)) == 9):
        assert n[i] == 2 and t[i].tolist() == [61, 61, 17 if e[i, 17] <= e[i, 61] else 61]
        assert np.abs(lp[i] + np.log(2)).max() <= 1e-6


def test_draws_follow_the_target(mri, gpu_ctx):
    """Speculative sampling leaves the target's distribution: the first token
    over 40000 trials against p (chi-square, 9 degrees of freedom, below 33.7:
    p-value 1e-4)."""
    import torch
    rng = np.random.default_rng(7)
    vocab, n = 10, 40000
    p = rng.dirichlet(np.ones(vocab))
    q = rng.dirichlet(np.ones(vocab))
    logits = np.zeros((n, 2, vocab), np.float32)
    logits[:, 0] = np.log(p)
    drafts = rng.choice(vocab, size=(n, 1), p=q).astype(np.int32)
    t, _, _ = mri.verify_draft(gpu(logits), gpu(drafts), gpu(rng.random((n, 1)).astype(np.float32)),
                               gpu(rng.exponential(1, (n, vocab)).astype(np.float32)),
                               draft_probs=gpu(np.broadcast_to(q.astype(np.float32), (n, 1, vocab))))
    seen = torch.bincount(t[:, 0].long(), minlength=vocab).cpu().numpy()
    assert (((seen - n * p) ** 2) / (n * p)).sum() < 33.7


def test_strided_inputs_and_streams(mri, gpu_ctx):
    import torch
    rng = np.random.default_rng(8)
    logits, drafts, u, e, q = inputs(rng, 3, 2, 300)
    want = mri.verify_draft(gpu(logits), gpu(drafts), gpu(u), gpu(e), draft_probs=gpu(q))
    wide = torch.zeros(3, 3, 600, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        view = wide[..., ::2]
        view.copy_(gpu(logits))
        got = mri.verify_draft(view, gpu(drafts), gpu(u), gpu(e), draft_probs=gpu(q))
        got = [t + 0 for t in got]
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(mri, gpu_ctx):
    import torch
    rng = np.random.default_rng(9)
    logits, drafts, u, e, q = (gpu(a) for a in inputs(rng, 2, 2, 50))
    with pytest.raises(mri.InvalidShape):
        mri.verify_draft(logits[0], drafts, u, e)
    with pytest.raises(mri.ShapeMismatch):
        mri.verify_draft(logits, drafts[:, :1], u, e)
    with pytest.raises(mri.ShapeMismatch):
        mri.verify_draft(logits, drafts, u, e[:, :-1])
    with pytest.raises(mri.ShapeMismatch):
        mri.verify_draft(logits, drafts, u, e, draft_probs=q[:, :1])
    with pytest.raises(mri.ShapeMismatch):
        mri.verify_draft(logits, drafts, u, e, temperature=torch.ones(3, device="cuda"))
    with pytest.raises(ValueError):
        mri.verify_draft(logits.cpu(), drafts, u, e)
    with pytest.raises(ValueError):
        mri.verify_draft(logits, drafts.long(), u, e)
    with pytest.raises(ValueError):
        mri.verify_draft(logits, drafts, u.double(), e)
    with pytest.raises(mri.InvalidShape):
        mri.verify_draft(torch.zeros(1, 66, 4, device="cuda"), torch.zeros(1, 65, dtype=torch.int32, device="cuda"),
                         torch.zeros(1, 65, device="cuda"), torch.ones(1, 4, device="cuda"))
    lib, h = gpu_ctx._lib, gpu_ctx.handle
    p = logits.data_ptr()
    assert lib.mri_verify_draft(None, p, p, p, p, None, None, 1, 1, 4, p, p, None) == 6
    assert lib.mri_verify_draft(h, None, p, p, p, None, None, 1, 1, 4, p, p, None) == 6
    assert lib.mri_verify_draft(h, p, None, p, p, None, None, 1, 1, 4, p, p, None) == 6
    assert lib.mri_verify_draft(h, p, p, p, p, None, None, 1, 1, 0, p, p, None) == 1


def test_overlapping_buffers(mri, gpu_ctx):
    """An output in an input's place is refused; a lone sequence's tokens may take its drafts' place."""
    import torch
    rng = np.random.default_rng(13)
    lib, h = gpu_ctx._lib, gpu_ctx.handle
    for b in (1, 3):
        logits, drafts, u, e, q = (gpu(a) for a in inputs(rng, b, 2, 5000))
        temp = torch.full((b,), 0.8, device="cuda")
        tokens, accepted, lp = mri.verify_draft(logits, drafts, u, e, draft_probs=q, temperature=temp)
        ins = [t.data_ptr() for t in (logits, drafts, u, e, q, temp)]
        room = torch.zeros(b * 3, dtype=torch.int32, device="cuda")
        room[:b * 2] = drafts.flatten()
        outs = [torch.zeros_like(t) for t in (tokens, accepted, lp)]

        def call(at=ins, out=[t.data_ptr() for t in outs]):
            return lib.mri_verify_draft(h, *at, b, 2, 5000, *out)

        torch.cuda.synchronize()
        launches = gpu_ctx.launch_count
        for i in range(3):
            for other in ins + [outs[(i + 1) % 3].data_ptr()]:
                out = [t.data_ptr() for t in outs]
                out[i] = other
                if not (b == 1 and i == 0 and other == ins[1]):
                    assert call(out=out) == 6, (b, i)
        assert call(out=[room.data_ptr() + 4] + [t.data_ptr() for t in outs[1:]], at=[ins[0], room.data_ptr()] + ins[2:]) == 6
        in_place = dict(out=[room.data_ptr()] + [t.data_ptr() for t in outs[1:]], at=[ins[0], room.data_ptr()] + ins[2:])
        if b > 1:
            assert call(**in_place) == 6
        assert gpu_ctx.launch_count == launches
        if b == 1:
            assert call(**in_place) == 0
            gpu_ctx.synchronize()
            assert torch.equal(room.view(1, 3), tokens) and torch.equal(outs[1], accepted) and torch.equal(outs[2], lp)
