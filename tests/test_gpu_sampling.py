"""Sampling on the GPU (kq_dec_sample) against its definition in 64 bits: the
tokens and the numbers of kept tokens are equal, the probability is within three
roundings of f32 (the weights' 2e-13 and their fixed point's 2^-45 lie far below):
2^-23 of itself."""
import math

import numpy as np
import pytest
import torch

from pesti_b200 import kq, sampling

pytestmark = pytest.mark.gpu

DEV = "cuda"


def chosen(z, t, k, p, m, u):
    """(token, probability, kept) of one row."""
    z = np.where(np.isnan(z), -np.inf, z.astype(np.float64))
    order = np.argsort(-z, kind="stable")
    order = order[z[order] > -np.inf]
    if not len(order):
        return -1, 0.0, 0
    top = z[order[0]]
    if not t > 0:
        order = order[:1]
    elif k > 0:
        order = order[:k]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp(np.where(z[order] == top, 0.0, (z[order] - top) / (t if t > 0 else 1.0)))
    n = len(order)
    if not p > 0:
        n = 1
    elif p < 1:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        n = max(1, int(np.count_nonzero(before < p * w.sum())))
    if not m <= 1:
        n = 1
    n = max(1, min(n, int(np.count_nonzero(w >= m))))
    order, w = order[:n], w[:n]
    up = np.argsort(order)
    order, w = order[up], w[up]
    run = np.cumsum(w)
    i = min(int(np.searchsorted(run, max(u, 0.0) * run[-1], side="right")), n - 1)
    return int(order[i]), w[i] / run[-1], n


def vec(x, b, dtype=torch.float32):
    return None if x is None else torch.tensor(np.broadcast_to(x, (b,)).copy(), dtype=dtype, device=DEV)


def check(ctx, logits, t=1.0, k=None, p=None, m=None, u=None, ref=None):
    """logits: numpy [B][V] or a CUDA tensor with its numpy form in `ref`."""
    z = ref if ref is not None else logits
    x = logits if ref is not None else torch.from_numpy(np.ascontiguousarray(logits, np.float32)).to(DEV)
    B = z.shape[0]
    rng = np.random.default_rng(B * z.shape[1])
    u = rng.random(B, dtype=np.float32) if u is None else np.broadcast_to(np.float32(u), (B,))
    td, kd, pd, md, ud = vec(t, B), vec(k, B, torch.int32), vec(p, B), vec(m, B), vec(u, B)
    got = []
    for _ in range(2):
        tok, prob = torch.full((B,), -9, dtype=torch.int32, device=DEV), torch.full((B,), -9.0, device=DEV)
        kept = torch.full((B,), -9, dtype=torch.int32, device=DEV)
        torch.cuda.synchronize()
        sampling.sample(ctx, x, ud, tok, temperature=td, top_k=kd, top_p=pd, min_p=md, prob=prob, kept=kept)
        ctx.synchronize()
        got.append((tok.cpu().numpy(), prob.cpu().numpy(), kept.cpu().numpy()))
    assert all(np.array_equal(a, b) for a, b in zip(*got))
    f = lambda v, d: np.broadcast_to(np.float32(d if v is None else v), (B,)).astype(np.float64)  # noqa: E731
    for b in range(B):
        want = chosen(z[b], f(t, 1)[b], int(np.broadcast_to(0 if k is None else k, (B,))[b]), f(p, 1)[b], f(m, 0)[b],
                      float(u[b]))
        tok, prob, kept = (int(got[0][0][b]), float(got[0][1][b]), int(got[0][2][b]))
        assert (tok, kept) == (want[0], want[2]), (b, tok, kept, want)
        assert abs(prob - want[1]) <= 2 ** -23 * want[1]
    return got[0]


SETTINGS = [dict(), dict(t=0.7, k=40), dict(t=0.8, p=0.9), dict(t=1.3, m=0.05), dict(t=0.9, k=50, p=0.95, m=0.02),
            dict(t=0.0), dict(t=2.5, k=700, p=0.8), dict(k=1500), dict(p=0.3), dict(t=5.0, p=0.99), dict(k=2, p=0.5),
            dict(t=0.5, k=512), dict(k=100, m=0.3)]


@pytest.mark.parametrize("vocab", [1, 2, 5, 33, 1000, 1024, 1025, 4097, 32000, 128256, 151936])
@pytest.mark.parametrize("setting", range(len(SETTINGS)))
def test_sampling(gpu_ctx, vocab, setting):
    rng = np.random.default_rng(vocab + setting)
    check(gpu_ctx, (2.5 * rng.standard_normal((3, vocab))).astype(np.float32), **SETTINGS[setting])


def test_every_row_has_settings_of_its_own(gpu_ctx):
    rng = np.random.default_rng(1)
    B = 70
    z = (2.0 * rng.standard_normal((B, 50257))).astype(np.float32)
    check(gpu_ctx, z, t=rng.choice([0.0, 0.6, 1.0, 1.5], B), k=rng.choice([0, 1, 20, 400, 900, 60000], B),
          p=rng.choice([0.0, 0.5, 0.9, 1.0, 2.0], B), m=rng.choice([0.0, 0.01, 0.2, 1.0, 1.5], B))


def test_the_largest_vocabulary_and_one_more(gpu_ctx):
    rng = np.random.default_rng(2)
    for setting in (dict(t=0.9, p=0.9), dict(k=50), dict()):
        check(gpu_ctx, (2.5 * rng.standard_normal((2, 393216))).astype(np.float32), **setting)
    x = torch.zeros((1, 393217), device=DEV)
    with pytest.raises(kq.KqError) as e:
        sampling.sample(gpu_ctx, x, torch.zeros(1, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV))
    assert e.value.status == kq.KQ_ERR_UNSUPPORTED


@pytest.mark.parametrize("setting", [dict(k=40), dict(p=0.9), dict(k=3000, p=0.7), dict(), dict(m=0.5), dict(k=600),
                                     dict(t=0.0), dict(k=40, p=0.5, m=0.1)])
def test_ties_go_to_the_lowest_index(gpu_ctx, setting):
    rng = np.random.default_rng(3)
    z = 2.0 * rng.standard_normal((4, 30000))
    z[0] = np.round(z[0])          # about ten values
    z[1] = np.round(z[1] * 16) / 16
    z[2] = 0.25                    # one value
    z[3] = np.where(rng.random(30000) < 0.5, 0.0, -0.0)
    check(gpu_ctx, z.astype(np.float32), **setting)


@pytest.mark.parametrize("setting", [dict(k=40), dict(p=0.9), dict(), dict(k=2000), dict(t=0.0), dict(m=0.1, p=0.95),
                                     dict(k=5, p=0.9)])
def test_masked_and_odd_logits(gpu_ctx, setting):
    rng = np.random.default_rng(4)
    z = (2.0 * rng.standard_normal((12, 5000))).astype(np.float32)
    z[0, 3:] = -np.inf                               # three tokens
    z[1] = -np.inf                                   # none
    z[2, rng.random(5000) < 0.9] = np.finfo(np.float32).min
    z[3, rng.random(5000) < 0.5] = np.nan
    z[4] = np.nan
    z[5, [7, 4000]] = np.inf                         # only these carry weight
    z[6] = np.finfo(np.float32).min
    z[7] *= 1e30
    z[8] *= 1e-30
    z[9] += 1e6
    z[10, :4999] = -np.inf
    z[11, 4321] = 3e38
    check(gpu_ctx, z, **setting)


@pytest.mark.parametrize("t", [1e-30, 1e-3, 1e3, 1e30, math.inf, math.nan, -1.0])
@pytest.mark.parametrize("setting", [dict(), dict(k=30), dict(p=0.6), dict(m=0.9)])
def test_extreme_temperatures(gpu_ctx, t, setting):
    rng = np.random.default_rng(5)
    check(gpu_ctx, rng.standard_normal((2, 3001)).astype(np.float32), t=t, **setting)


@pytest.mark.parametrize("u", [0.0, 1e-30, 0.5, 1 - 2 ** -24, 1.0, 7.0, -1.0, math.nan])
def test_random_numbers_at_their_borders(gpu_ctx, u):
    rng = np.random.default_rng(6)
    z = rng.standard_normal((2, 2000)).astype(np.float32)
    uu = 0.0 if math.isnan(u) else u
    want = check(gpu_ctx, z, u=uu)[0], check(gpu_ctx, z, k=10, u=uu)[0]
    for kw, w in zip((dict(), dict(top_k=vec(10, 2, torch.int32))), want):
        tok = torch.zeros(2, dtype=torch.int32, device=DEV)
        x, ud = torch.from_numpy(z).to(DEV), vec(u, 2)
        torch.cuda.synchronize()
        sampling.sample(gpu_ctx, x, ud, tok, **kw)
        gpu_ctx.synchronize()
        assert tok.tolist() == w.tolist()


@pytest.mark.parametrize("peak", [0.0, 5.0, 12.0, 40.0])
def test_one_token_above_a_flat_rest(gpu_ctx, peak):
    """The border of the nucleus lies among thousands of tokens of nearly the same weight."""
    rng = np.random.default_rng(7)
    z = (1e-3 * rng.standard_normal((4, 60000))).astype(np.float32)
    z[:, 12345] += peak
    check(gpu_ctx, z, p=np.array([0.1, 0.5, 0.9, 0.999]))
    check(gpu_ctx, z, m=np.array([0.5, 1e-4, 1e-17, 1e-20]))


def test_draws_follow_the_weights(gpu_ctx):
    """1000 evenly spaced numbers over one row: each token as often as its share of them says."""
    rng = np.random.default_rng(8)
    row = rng.standard_normal(50).astype(np.float32)
    n = 1000
    u = (np.arange(n, dtype=np.float32) + 0.5) / n
    tok = check(gpu_ctx, np.tile(row, (n, 1)), u=u)[0]
    share = np.exp(row.astype(np.float64))
    share /= share.sum()
    assert np.abs(np.bincount(tok, minlength=50) - n * share).max() <= 1.0


@pytest.mark.parametrize("shift,extra", [(0, 0), (1, 0), (0, 3), (3, 5)])
def test_rows_of_any_alignment(gpu_ctx, shift, extra):
    rng = np.random.default_rng(9)
    vocab = 20001
    wide = torch.from_numpy((2 * rng.standard_normal((5, vocab + shift + extra))).astype(np.float32)).to(DEV)
    x = wide[:, shift:shift + vocab]
    for s in (dict(k=20), dict(p=0.8), dict()):
        check(gpu_ctx, x, ref=x.cpu().numpy(), **s)


def test_captured_draws_follow_the_numbers_of_the_moment(gpu_ctx):
    rng = np.random.default_rng(10)
    z = rng.standard_normal((3, 9000)).astype(np.float32)
    x, u, p = torch.from_numpy(z).to(DEV), vec(0.0, 3), vec(0.9, 3)
    tok = torch.zeros(3, dtype=torch.int32, device=DEV)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    gpu_ctx.set_stream(stream)
    try:
        sampling.sample(gpu_ctx, x, u, tok, top_p=p)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            sampling.sample(gpu_ctx, x, u, tok, top_p=p)
        for v in (0.1, 0.5, 0.93):
            with torch.cuda.stream(stream):
                u.fill_(v)
                g.replay()
            gpu_ctx.synchronize()
            assert tok.tolist() == [chosen(z[b], 1.0, 0, float(np.float32(0.9)), 0.0, float(np.float32(v)))[0]
                                    for b in range(3)]
        del g
    finally:
        gpu_ctx.set_stream(None)


def test_refusals(gpu_ctx):
    f, i = torch.zeros(2, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    x = torch.zeros((2, 8), device=DEV)
    for a in ((x.half(), f, i), (x.t(), f, i), (x, f[:1], i), (x, f, f), (x, f.cpu(), i), (x[:, :0], f, i), (x, None, i)):
        with pytest.raises(kq.KqError) as e:
            sampling.sample(gpu_ctx, *a)
        assert e.value.status == kq.KQ_ERR_INVALID_ARG
    for kw in (dict(temperature=i), dict(top_k=f), dict(top_p=f[:1]), dict(min_p=f.double()), dict(prob=i), dict(kept=f)):
        with pytest.raises(kq.KqError) as e:
            sampling.sample(gpu_ctx, x, f, i, **kw)
        assert e.value.status == kq.KQ_ERR_INVALID_ARG
