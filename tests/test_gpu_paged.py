"""The paged key-value cache on the GPU (kq_kv_*) against a plain 64-bit
implementation: append, attention of one token per sequence with and without the
rotation, and eviction by accumulated attention weight.

Tolerances.  Attention: a score's error is at most sum |q_i k_i| / sqrt(hd) (about
11 at 128 and 15 at 256 normal values) times 2^-22 for q's two f16 parts and 4 x
2^-23 for the products' cut-off sums, below 1.1e-5; the weights' relative error is
that, and an output's, over the largest |v|, at most twice it: 2e-5.  Rotation:
(|x| + |y|) times pi 2^-25 for the angle, 2 ulp for sine and cosine and three
roundings, below 7e-7 of the largest value: 1e-6.  A cached f16 value adds half a
step, 2^-11 of itself (2^-25 below the normal range)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from pesti_b200 import decoder as dec
from pesti_b200 import kq, paged

pytestmark = pytest.mark.gpu

TOL_OUT, TOL_TURN = 2e-5, 1e-6
DEV = "cuda"


def turn(x, pos, theta):
    """Rows x [n][heads][hd] turned to pos [n], in 64 bits."""
    half = x.shape[-1] // 2
    freq = theta ** (-torch.arange(half, dtype=torch.float64, device=x.device) / half)
    angle = pos.double()[:, None, None] * freq
    a, b = x[..., :half].double(), x[..., half:].double()
    c, s = torch.cos(angle), torch.sin(angle)
    return torch.cat([a * c - b * s, a * s + b * c], -1)


class Setup:
    """Pools, block table and lengths; everything that no sequence uses is NaN or out of range."""

    def __init__(self, ctx, lens, hq, hkv, hd, page, seed=0, spare=3, k=None, v=None, width=None):
        self.ctx, self.hq, self.hkv, self.hd, self.page, self.lens_h = ctx, hq, hkv, hd, page, lens
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        self.g = g
        blocks = [-(-n // page) for n in lens]
        self.pages = sum(blocks) + spare
        order = torch.randperm(self.pages, generator=g, device=DEV).int().cpu()
        width = width or max(max(blocks), 1) + 1
        table = torch.full((len(lens), width), 2 ** 31 - 1, dtype=torch.int32)
        table[:, -1] = -7
        at = 0
        for b, n in enumerate(blocks):
            table[b, :n] = order[at:at + n]
            at += n
        self.table = table.to(DEV)
        shape = (self.pages, hkv, page, hd)
        self.k = torch.empty(shape, dtype=torch.float16, device=DEV) if k is None else k
        self.v = torch.empty(shape, dtype=torch.float16, device=DEV) if v is None else v
        for pool in (self.k, self.v):
            pool.copy_(torch.randn(shape, generator=g, device=DEV))
        used = torch.zeros((self.pages, page), dtype=torch.bool, device=DEV)
        for b, n in enumerate(lens):
            for j in range(blocks[b]):
                used[int(table[b, j]), :min(page, n - j * page)] = True
        for pool in (self.k, self.v):
            pool.masked_fill_(~used[:, None, :, None], float("nan"))
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.cache = paged.PagedCache(ctx, self.k, self.v)

    def rows(self, pool, b, h, n):
        ids = self.table[b, :-(-n // self.page)].long()
        return pool[ids, h].reshape(-1, self.hd)[:n].double()

    def reference(self, q):
        """q [B][hq][hd] -> out [B][hq][hd] and the summed weights per (sequence, kv head)."""
        G = self.hq // self.hkv
        out, mass = torch.zeros(q.shape, dtype=torch.float64, device=DEV), {}
        for b, n in enumerate(self.lens_h):
            for h in range(self.hkv if n else 0):
                k, v = self.rows(self.k, b, h, n), self.rows(self.v, b, h, n)
                p = torch.softmax(q[b, h * G:(h + 1) * G].double() @ k.T / math.sqrt(self.hd), -1)
                out[b, h * G:(h + 1) * G] = p @ v
                mass[b, h] = p.sum(0)
        return out, mass


def far(out, ref, scale):
    assert torch.isfinite(out).all()
    return float((out.double() - ref).abs().max()) / scale


RAGGED = [130, 0, 1, 16, 17, 63, 64, 65, 200, 127, 128, 129, 3, 0, 500, 1, 31]
ATTENTION = [
    # hd, hq, hkv, page, lens
    (128, 32, 8, 64, [2049]),
    (128, 32, 8, 16, RAGGED),
    (64, 14, 2, 32, RAGGED * 3),
    (64, 4, 4, 48, [1000, 7, 0]),
    (256, 8, 4, 64, RAGGED),
    (256, 3, 1, 16, [40000, 1]),
    (128, 1, 1, 1024, [70001]),
    (128, 9, 1, 64, RAGGED),
    (128, 32, 2, 128, [5000, 0, 77, 1]),
    (64, 26, 2, 64, RAGGED),
    (256, 16, 1, 112, [3000, 63, 0, 1]),
    (64, 7, 7, 256, [0, 0, 1]),
    (128, 64, 8, 64, [64] * 70),
    (128, 8, 8, 16, [1] * 300),
    (128, 12, 4, 64, [100000, 5, 300]),
]


@pytest.mark.parametrize("hd,hq,hkv,page,lens", ATTENTION)
@pytest.mark.parametrize("mass", [False, True])
def test_attention(gpu_ctx, hd, hq, hkv, page, lens, mass):
    s = Setup(gpu_ctx, lens, hq, hkv, hd, page, seed=hd + hq + page)
    B = len(lens)
    q = 1.5 * torch.randn((B, hq * hd), generator=s.g, device=DEV)
    ref, ref_mass = s.reference(q.view(B, hq, hd))
    ld = max(max(lens), 1) + 2
    scratch = s.cache.scratch(B, hq, ld if mass else 0)
    outs, masses = [], []
    for _ in range(2):  # the second call finds the counters at zero
        out = torch.full((B, hq * hd), float("nan"), device=DEV)
        m = torch.full((B, hkv, ld), 0.25, device=DEV) if mass else None
        torch.cuda.synchronize()
        s.cache.attention(q, s.table, s.lens, out, scratch, mass=m)
        gpu_ctx.synchronize()
        outs.append(out)
        masses.append(m)
    assert torch.equal(outs[0], outs[1])
    vmax = float(s.v.nan_to_num(0).abs().max())
    assert far(outs[0].view(B, hq, hd), ref, vmax) <= TOL_OUT
    for b, n in enumerate(lens):
        if n == 0:
            assert not outs[0][b].any()
    if mass:
        assert torch.equal(masses[0], masses[1])
        want = torch.full((B, hkv, ld), 0.25, dtype=torch.float64, device=DEV)
        for (b, h), m in ref_mass.items():
            want[b, h, :len(m)] += m
        # a weight's relative error is TOL_OUT / 2 at most, the sum over a group G times that
        G = hq // hkv
        assert float((masses[0].double() - want).abs().max()) <= TOL_OUT * G + 2 ** -24 * (G + 1)
        for b, n in enumerate(lens):
            assert (masses[0][b, :, n:] == 0.25).all()


@pytest.mark.parametrize("hd,hq,hkv,page,lens", [c for c in ATTENTION if max(c[4]) < 50000])
def test_rope_attention(gpu_ctx, hd, hq, hkv, page, lens):
    theta = 500000.0
    s = Setup(gpu_ctx, lens, hq, hkv, hd, page, seed=hd + hq)
    B = len(lens)
    qkv = 1.5 * torch.randn((B, (hq + 2 * hkv) * hd), generator=s.g, device=DEV)
    keep = qkv.clone()
    pos = (s.lens - 1 + torch.randint(0, 120000, (B,), generator=s.g, device=DEV)).int()
    ld = max(max(lens), 1)
    mass = torch.rand((B, hkv, ld), generator=s.g, device=DEV)
    mass0, spos = mass.clone(), torch.full((B, hkv, ld), -3, dtype=torch.int32, device=DEV)
    for b, n in enumerate(lens):  # the new slot's row is not there yet
        if n:
            page_id = int(s.table[b, (n - 1) // page])
            s.k[page_id, :, (n - 1) % page] = float("nan")
            s.v[page_id, :, (n - 1) % page] = float("nan")
    k0, v0 = s.k.clone(), s.v.clone()
    out = torch.full((B, hq * hd), float("nan"), device=DEV)
    scratch = s.cache.scratch(B, hq, ld)
    torch.cuda.synchronize()
    s.cache.rope_attention(qkv, s.table, s.lens, out, scratch, theta=theta, pos=pos, mass=mass, slot_pos=spos)
    gpu_ctx.synchronize()
    assert torch.equal(qkv, keep)
    rows = qkv.view(B, hq + 2 * hkv, hd)
    turned = turn(rows[:, :hq + hkv], pos, theta)
    top = float(rows.abs().max())
    for b, n in enumerate(lens):
        if not n:
            continue
        page_id, r = int(s.table[b, (n - 1) // page]), (n - 1) % page
        k, v = s.k[page_id, :, r], s.v[page_id, :, r]
        want = turned[b, hq:]
        assert ((k.double() - want).abs() <= TOL_TURN * top + 2 ** -11 * want.abs() + 2 ** -25).all()
        assert torch.equal(v, rows[b, hq + hkv:].half())
        k0[page_id, :, r], v0[page_id, :, r] = k, v
        assert (spos[b, :, n - 1] == pos[b]).all() and (spos[b, :, :n - 1] == -3).all()
    assert torch.equal(s.k.nan_to_num(7), k0.nan_to_num(7)) and torch.equal(s.v.nan_to_num(7), v0.nan_to_num(7))
    ref, ref_mass = s.reference(turned[:, :hq])
    # the turned q is off by TOL_TURN of its largest value more: a score by sqrt(hd) sum |k| of that at most
    slack = 2 * TOL_TURN * top * math.sqrt(hd)
    assert far(out.view(B, hq, hd), ref, float(s.v.nan_to_num(0).abs().max())) <= TOL_OUT + slack
    for (b, h), m in ref_mass.items():
        n = len(m)
        want = mass0[b, h, :n].double() + m
        want[n - 1] = m[n - 1]
        assert float((mass[b, h, :n].double() - want).abs().max()) <= (TOL_OUT + slack) * (hq // hkv) + 1e-6
        assert torch.equal(mass[b, h, n:], mass0[b, h, n:])


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_the_appended_key_is_the_exact_one_rounded(gpu_ctx, hd):
    """k is turned in 64 bits, to 1e-10 of its length, rounded to f32 and that to f16 (as torch
    converts a double): the first rounding moves at about 1e-3 of the elements, which moves the
    second at 1e-4 of those, where sums in f32 would at 2e-4 of all."""
    B, hq, hkv, theta = 64 * 256 // hd, 4, 4, 1e6
    s = Setup(gpu_ctx, [3] * B, hq, hkv, hd, 16, seed=hd)
    qkv = torch.randn((B, (hq + 2 * hkv) * hd), generator=s.g, device=DEV)
    pos = torch.randint(0, 120000, (B,), generator=s.g, device=DEV).int()
    out = torch.zeros((B, hq * hd), device=DEV)
    torch.cuda.synchronize()
    s.cache.rope_attention(qkv, s.table, s.lens, out, s.cache.scratch(B, hq, 0), theta=theta, pos=pos)
    gpu_ctx.synchronize()
    want = turn(qkv.view(B, hq + 2 * hkv, hd)[:, hq:hq + hkv], pos, theta).half()
    assert int((s.k[s.table[:, 0].long(), :, 2] != want).sum()) <= 2  # of 65,536


def test_default_positions_and_the_contiguous_cache_agree(gpu_ctx):
    """Pages in order are the contiguous cache: kq_dec_rope_attention's own result."""
    hd, hq, hkv, B, pos, page = 128, 32, 8, 3, 300, 16
    lib, max_seq = dec._bind(gpu_ctx.lib), 320
    g = torch.Generator(device=DEV)
    g.manual_seed(4)
    k = torch.randn((B, hkv, max_seq, hd), generator=g, device=DEV).half()
    v = torch.randn((B, hkv, max_seq, hd), generator=g, device=DEV).half()
    kp, vp = (t.view(B, hkv, max_seq // page, page, hd).transpose(1, 2).reshape(-1, hkv, page, hd).contiguous()
              for t in (k, v))
    qkv = torch.randn((B, (hq + 2 * hkv) * hd), generator=g, device=DEV)
    out, out2 = (torch.empty((B, hq * hd), device=DEV) for _ in range(2))
    n = lib.kq_dec_attention_scratch(gpu_ctx.handle, B, hq, hkv, hd, max_seq)
    old = torch.zeros(n // 4, device=DEV)
    P = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    torch.cuda.synchronize()
    gpu_ctx.check(lib.kq_dec_rope_attention(gpu_ctx.handle, P(qkv), qkv.shape[1], P(k), P(v), P(out), hq * hd, B, hq,
                                            hkv, hd, pos, max_seq, 5e5, P(old), n), "kq_dec_rope_attention")
    table = torch.arange(B * max_seq // page, dtype=torch.int32, device=DEV).view(B, -1)
    cache = paged.PagedCache(gpu_ctx, kp, vp)
    scratch = cache.scratch(B, hq)
    lens = torch.full((B,), pos + 1, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    cache.rope_attention(qkv, table, lens, out2, scratch, theta=5e5)
    gpu_ctx.synchronize()
    # the older kernel's f32 angles are off by 2^-24 of 300 radians, its cached keys by a step more
    assert float((out - out2).abs().max()) <= 1e-3 * float(out.abs().max())
    assert torch.equal(vp.view(B, -1, hkv, page, hd).transpose(1, 2).reshape(v.shape), v)


def test_strided_rows_and_pools(gpu_ctx):
    """K and V of a page side by side in one tensor, query and output rows inside wider ones."""
    hd, hq, hkv, page, lens = 128, 12, 4, 32, [70, 0, 33, 400]
    both = torch.empty((40, 2, hkv, page, hd), dtype=torch.float16, device=DEV)
    s = Setup(gpu_ctx, lens, hq, hkv, hd, page, k=both[:sum(-(-n // page) for n in lens) + 3, 0],
              v=both[:sum(-(-n // page) for n in lens) + 3, 1])
    wide = torch.randn((4, hq * hd + 7), device=DEV)
    q = wide[:, 3:3 + hq * hd]  # not 16-byte aligned, odd row stride
    outw = torch.full((4, hq * hd + 5), 9.0, device=DEV)
    out = outw[:, 1:1 + hq * hd]
    scratch = s.cache.scratch(4, hq)
    torch.cuda.synchronize()
    s.cache.attention(q, s.table, s.lens, out, scratch)
    gpu_ctx.synchronize()
    ref, _ = s.reference(q.reshape(4, hq, hd))
    assert far(out.reshape(4, hq, hd), ref, float(s.v.nan_to_num(0).abs().max())) <= TOL_OUT
    assert (outw[:, 0] == 9).all() and (outw[:, 1 + hq * hd:] == 9).all()


def test_pages_past_32_bits(gpu_ctx):
    """Rows behind 2^32 elements of the pools."""
    hd, hq, hkv, page = 128, 8, 8, 64
    pages = (1 << 32) // (hkv * page * hd) + 40
    k, v = (torch.empty((pages, hkv, page, hd), dtype=torch.float16, device=DEV) for _ in range(2))
    ids = [pages - 1, 2, pages - 17]
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    for i in ids:
        k[i], v[i] = (torch.randn(k[i].shape, generator=g, device=DEV).half() for _ in range(2))
    cache = paged.PagedCache(gpu_ctx, k, v)
    table = torch.tensor([ids], dtype=torch.int32, device=DEV)
    n = 2 * page + 10
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    qkv = torch.randn((1, 3 * 8 * hd), generator=g, device=DEV)
    out = torch.empty((1, hq * hd), device=DEV)
    scratch = cache.scratch(1, hq)
    torch.cuda.synchronize()
    cache.rope_attention(qkv, table, lens, out, scratch, theta=1e4)
    gpu_ctx.synchronize()
    rows = qkv.view(1, 24, hd)
    pos = lens - 1
    q = turn(rows[:, :8], pos, 1e4)[0]
    assert torch.equal(v[ids[2], :, 9], rows[0, 16:].half())
    kk, vv = (t[ids].transpose(0, 1).reshape(hkv, -1, hd)[:, :n].double() for t in (k, v))
    p = torch.softmax(torch.einsum("hd,hnd->hn", q, kk) / math.sqrt(hd), -1)
    ref = torch.einsum("hn,hnd->hd", p, vv)
    assert far(out.view(hq, hd), ref, float(vv.abs().max())) <= TOL_OUT + 1e-5
    # eviction moves rows between far pages: keep the last 100 positions
    mass = torch.rand((1, hkv, n), generator=g, device=DEV)
    spos = torch.arange(n, dtype=torch.int32, device=DEV).expand(1, hkv, n).contiguous()
    want = kk[:, n - 100:].clone()
    since = torch.tensor([n - 100], dtype=torch.int32, device=DEV)
    es = cache.evict_scratch(1, n)
    torch.cuda.synchronize()
    cache.evict(table, lens, lens, mass, spos, mass, spos, 100, es, recent_from=since)
    gpu_ctx.synchronize()
    assert lens.tolist() == [100]
    got = k[ids].transpose(0, 1).reshape(hkv, -1, hd)[:, :100].double()
    order = spos[0, :, :100].long() - (n - 100)
    for h in range(hkv):
        assert sorted(order[h].tolist()) == list(range(100))
        assert torch.equal(got[h], want[h][order[h]])
    del k, v, cache
    torch.cuda.empty_cache()


def test_one_scratch_serves_calls_of_other_sizes(gpu_ctx):
    a = Setup(gpu_ctx, [900, 3, 70] * 8, 32, 8, 128, 64, seed=1)
    b = Setup(gpu_ctx, [5000], 16, 1, 64, 16, seed=2)
    scratch = max((a.cache.scratch(24, 32, 900), b.cache.scratch(1, 16, 0)), key=lambda t: t.numel())
    qa, qb = torch.randn((24, 32 * 128), device=DEV), torch.randn((1, 16 * 64), device=DEV)
    oa, ob = torch.empty_like(qa), torch.empty_like(qb)
    m = torch.zeros((24, 8, 900), device=DEV)
    ra, rb = a.reference(qa.view(24, 32, 128))[0], b.reference(qb.view(1, 16, 64))[0]
    torch.cuda.synchronize()
    for _ in range(3):
        a.cache.attention(qa, a.table, a.lens, oa, scratch, mass=m)
        b.cache.attention(qb, b.table, b.lens, ob, scratch)
        a.cache.attention(qa[:1], a.table[:1], a.lens[:1], oa[:1], scratch)
    gpu_ctx.synchronize()
    assert far(oa.view(24, 32, 128), ra, 5) <= TOL_OUT and far(ob.view(1, 16, 64), rb, 5) <= TOL_OUT


def test_captured_calls_follow_the_lengths_of_the_moment(gpu_ctx):
    hd, hq, hkv, page = 64, 14, 2, 16
    s = Setup(gpu_ctx, [600, 40, 0, 5], hq, hkv, hd, page, seed=9)
    qkv = torch.randn((4, (hq + 2 * hkv) * hd), generator=s.g, device=DEV)
    q = torch.randn((4, hq * hd), generator=s.g, device=DEV)
    out, out2 = torch.empty((4, hq * hd), device=DEV), torch.empty((4, hq * hd), device=DEV)
    scratch = s.cache.scratch(4, hq)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    gpu_ctx.set_stream(stream)
    try:
        s.cache.attention(q, s.table, s.lens, out, scratch)
        graphs = []
        for fn in (lambda: s.cache.attention(q, s.table, s.lens, out, scratch),
                   lambda: s.cache.rope_attention(qkv, s.table, s.lens, out2, scratch, theta=1e4)):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                fn()
            graphs.append(g)
        for lens in ([600, 40, 0, 5], [1, 0, 0, 5], [599, 40, 0, 1], [0, 0, 0, 0]):
            s.lens_h = lens
            with torch.cuda.stream(stream):
                s.lens.copy_(torch.tensor(lens, dtype=torch.int32))
                graphs[0].replay()
            gpu_ctx.synchronize()
            ref, _ = s.reference(q.view(4, hq, hd))
            assert far(out.view(4, hq, hd), ref, 5) <= TOL_OUT
            with torch.cuda.stream(stream):
                graphs[1].replay()  # appends, so the rows change
            gpu_ctx.synchronize()
            ref, _ = s.reference(turn(qkv.view(4, -1, hd)[:, :hq], s.lens - 1, 1e4))
            assert far(out2.view(4, hq, hd), ref, 5) <= TOL_OUT + 1e-5
        del graphs, g
    finally:
        gpu_ctx.set_stream(None)


def test_shared_pages_are_read_by_every_sequence(gpu_ctx):
    s = Setup(gpu_ctx, [200, 200], 8, 2, 128, 64, seed=3)
    s.table[1, :2] = s.table[0, :2]  # a common prefix of two pages
    q = torch.randn((2, 8 * 128), generator=s.g, device=DEV)
    out = torch.empty_like(q)
    scratch = s.cache.scratch(2, 8)
    torch.cuda.synchronize()
    s.cache.attention(q, s.table, s.lens, out, scratch)
    gpu_ctx.synchronize()
    assert far(out.view(2, 8, 128), s.reference(q.view(2, 8, 128))[0], 5) <= TOL_OUT


# ---- append -----------------------------------------------------------------------------


@pytest.mark.parametrize("hd,hq,hkv,page", [(128, 32, 8, 64), (64, 14, 2, 16), (256, 5, 5, 48), (64, 1, 1, 16)])
@pytest.mark.parametrize("shift", [0, 1])  # 1: rows that are not 16-byte aligned
def test_append(gpu_ctx, hd, hq, hkv, page, shift):
    theta, n, B = 1e6, 75, 3
    s = Setup(gpu_ctx, [200, 90, 17], hq, hkv, hd, page, seed=5)
    cols = (hq + 2 * hkv) * hd
    qkv = torch.randn((n, cols + 3 * shift), generator=s.g, device=DEV)[:, shift:shift + cols]
    rng = np.random.default_rng(hd)
    cells = [(b, t) for b, m in enumerate(s.lens_h) for t in range(m)]
    pick = [cells[i] for i in rng.permutation(len(cells))[:n]]
    seqs = torch.tensor([p[0] for p in pick], dtype=torch.int32, device=DEV)
    slots = torch.tensor([p[1] if i % 7 else -1 for i, p in enumerate(pick)], dtype=torch.int32, device=DEV)
    pos = torch.tensor(rng.integers(0, 130000, n), dtype=torch.int32, device=DEV)
    q_out = torch.full((n, hq * hd + shift), 5.0, device=DEV)
    spos = torch.full((B, hkv, 256), -1, dtype=torch.int32, device=DEV)
    k0, v0 = s.k.clone(), s.v.clone()
    torch.cuda.synchronize()
    s.cache.append(qkv, s.table, slots, theta=theta, seqs=seqs, pos=pos, q_out=q_out, slot_pos=spos)
    gpu_ctx.synchronize()
    rows = qkv.reshape(n, hq + 2 * hkv, hd)
    turned = turn(rows[:, :hq + hkv], pos, theta)
    top = float(rows.abs().max())
    for i, (b, t) in enumerate(pick):
        if slots[i] < 0:
            assert (q_out[i] == 5).all()
            continue
        want = turned[i].reshape(-1)
        assert float((q_out[i, :hq * hd].double() - want[:hq * hd]).abs().max()) <= TOL_TURN * top
        at, r = int(s.table[b, t // page]), t % page
        want = turned[i, hq:]
        assert ((s.k[at, :, r].double() - want).abs() <= TOL_TURN * top + 2 ** -11 * want.abs() + 2 ** -25).all()
        assert torch.equal(s.v[at, :, r], rows[i, hq + hkv:].half())
        assert (spos[b, :, t] == pos[i]).all()
        k0[at, :, r], v0[at, :, r] = s.k[at, :, r], s.v[at, :, r]
    assert torch.equal(s.k.nan_to_num(7), k0.nan_to_num(7)) and torch.equal(s.v.nan_to_num(7), v0.nan_to_num(7))
    assert int((spos >= 0).sum()) == hkv * int((slots >= 0).sum())


def test_append_in_place_and_defaults(gpu_ctx):
    """q_out may be qkv itself; row r is sequence r at position slots[r] by default; no q wanted."""
    hd, hq, hkv = 128, 6, 2
    s = Setup(gpu_ctx, [40, 50, 1], hq, hkv, hd, 16, seed=6)
    qkv = torch.randn((3, (hq + 2 * hkv) * hd), generator=s.g, device=DEV)
    slots = torch.tensor([39, 7, 0], dtype=torch.int32, device=DEV)
    want = turn(qkv.view(3, -1, hd)[:, :hq], slots, 1e4)
    rest = qkv[:, hq * hd:].clone()
    k1, v1 = s.k.clone(), s.v.clone()
    c1 = paged.PagedCache(gpu_ctx, k1, v1)
    torch.cuda.synchronize()
    c1.append(qkv, s.table, slots, theta=1e4)
    s.cache.append(qkv[:1], s.table, slots[:1], theta=1e4, q_out=qkv[:1, :hq * hd])
    s.cache.append(qkv[1:], s.table[1:], slots[1:], theta=1e4, q_out=qkv[1:])
    gpu_ctx.synchronize()
    assert float((qkv[:, :hq * hd].view(3, hq, hd).double() - want).abs().max()) <= TOL_TURN * float(want.abs().max()) * 2
    assert torch.equal(qkv[:, hq * hd:], rest)
    assert torch.equal(k1.nan_to_num(7), s.k.nan_to_num(7))


def test_many_rows(gpu_ctx):
    """More rows than fit one wave, in one sequence of many pages."""
    hd, hq, hkv, n = 64, 3, 1, 9001
    s = Setup(gpu_ctx, [n], hq, hkv, hd, 16, seed=7)
    qkv = torch.randn((n, 5 * hd), generator=s.g, device=DEV)
    slots = torch.arange(n, dtype=torch.int32, device=DEV)
    q_out, seqs = torch.empty((n, hq * hd), device=DEV), torch.zeros_like(slots)
    torch.cuda.synchronize()
    s.cache.append(qkv, s.table, slots, theta=1e4, seqs=seqs, q_out=q_out)
    gpu_ctx.synchronize()
    t = turn(qkv.view(n, 5, hd)[:, :4], slots, 1e4)
    top = float(qkv.abs().max())
    assert float((q_out.view(n, hq, hd).double() - t[:, :3]).abs().max()) <= TOL_TURN * top
    assert torch.equal(s.rows(s.v, 0, 0, n).half(), qkv[:, 4 * hd:].half())
    assert float((s.rows(s.k, 0, 0, n) - t[:, 3]).abs().max()) <= TOL_TURN * top + 2 ** -11 * 2 * top


# ---- eviction -----------------------------------------------------------------------------


def keep_of(mass, spos, since, keep):
    """What stays of one head's slots: new slot -> old slot."""
    n = len(mass)
    if n <= keep:
        return np.arange(n)
    m = np.where(np.isnan(mass), -np.inf, mass.astype(np.float64))
    first = spos >= since
    order = sorted(range(n), key=lambda i: (not first[i], 0.0 if first[i] else -m[i], i))
    stay = np.zeros(n, bool)
    stay[order[:keep]] = True
    src = np.arange(keep)
    src[~stay[:keep]] = np.nonzero(stay[keep:])[0] + keep
    return src


def values(kind, shape, rng):
    if kind == "ties":
        return rng.integers(0, 3, shape).astype(np.float32)
    if kind == "equal":
        return np.full(shape, 0.5, np.float32)
    m = np.exp(2 * rng.standard_normal(shape)).astype(np.float32)
    if kind == "odd":
        u = rng.random(shape)
        for lo, x in ((0.0, np.nan), (0.05, np.inf), (0.1, -np.inf), (0.15, -0.0), (0.25, 0.0), (0.35, -1.5), (0.4, 1e-42)):
            m[(u >= lo) & (u < lo + (0.1 if x == 0 else 0.05))] = x
    return m


@pytest.mark.parametrize("hd,hkv,page,lens,keep,recent,kind", [
    (128, 8, 64, [300, 100, 0, 101, 1, 99], 100, 20, "plain"),
    (128, 8, 64, [300, 100, 0, 101, 1, 99], 100, 100, "ties"),
    (64, 2, 16, [2113] * 5, 2048, 256, "plain"),
    (64, 3, 16, [500, 37], 1, 0, "ties"),
    (64, 1, 48, [1500], 700, 0, "equal"),
    (256, 2, 64, [777, 600], 300, 50, "odd"),
    (128, 2, 64, [4097, 5000], 4096, 5000, "plain"),   # more protected than stay
    (64, 1, 64, [40960, 40961, 50], 20000, 64, "ties"),
    (64, 1, 256, [100003], 5000, 300, "odd"),
    (64, 1, 256, [100003], 99000, 0, "plain"),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_eviction(gpu_ctx, hd, hkv, page, lens, keep, recent, kind, in_place):
    B, ld = len(lens), max(lens) + 1
    s = Setup(gpu_ctx, lens, hkv, hkv, hd, page, seed=keep)
    rng = np.random.default_rng(keep + B)
    mass = values(kind, (B, hkv, ld), rng)
    spos = np.stack([np.stack([rng.permutation(ld) for _ in range(hkv)]) for _ in range(B)]).astype(np.int32)
    since = np.array([ld - recent] * B, np.int32)
    k0, v0 = s.k.clone(), s.v.clone()
    m, p = torch.from_numpy(mass).to(DEV), torch.from_numpy(spos).to(DEV)
    mo, po = (m, p) if in_place else (torch.full_like(m, 77.0), torch.full_like(p, -77))
    before = mo.clone()
    lens_out = s.lens if in_place else torch.zeros_like(s.lens)
    scratch = s.cache.evict_scratch(B, ld).fill_(255)
    recent_from = torch.from_numpy(since).to(DEV) if recent else None
    torch.cuda.synchronize()
    s.cache.evict(s.table, s.lens, lens_out, m, p, mo, po, keep, scratch, recent_from=recent_from)
    gpu_ctx.synchronize()
    assert lens_out.tolist() == [min(n, keep) for n in lens]
    for b, n in enumerate(lens):
        for h in range(hkv):
            src = keep_of(mass[b, h, :n], spos[b, h, :n], since[b] if recent else 1 << 40, keep)
            assert np.array_equal(mo[b, h, :len(src)].cpu().numpy(), mass[b, h, src], equal_nan=True)
            assert np.array_equal(po[b, h, :len(src)].cpu().numpy(), spos[b, h, src])
            assert torch.equal(mo[b, h, len(src):].nan_to_num(3), before[b, h, len(src):].nan_to_num(3))
            if len(src):
                for pool, old in ((s.k, k0), (s.v, v0)):
                    assert torch.equal(s.rows(pool, b, h, len(src)), s.rows(old, b, h, n)[torch.from_numpy(src).to(DEV)])


def test_eviction_keeps_the_attention_of_what_stays(gpu_ctx):
    """Weights gathered by the attention itself; afterwards the output is that over the kept slots."""
    hd, hq, hkv, page, lens, keep = 128, 16, 4, 32, [500, 64, 129], 64
    s = Setup(gpu_ctx, lens, hq, hkv, hd, page, seed=11)
    B, ld = 3, 512
    q = 2.0 * torch.randn((B, hq * hd), generator=s.g, device=DEV)
    out, mass = torch.empty_like(q), torch.zeros((B, hkv, ld), device=DEV)
    spos = torch.arange(ld, dtype=torch.int32, device=DEV).expand(B, hkv, ld).contiguous()
    scratch, es = s.cache.scratch(B, hq, ld), s.cache.evict_scratch(B, ld)
    kv = {(b, h): (s.rows(s.k, b, h, n), s.rows(s.v, b, h, n)) for b, n in enumerate(lens) for h in range(hkv)}
    torch.cuda.synchronize()
    s.cache.attention(q, s.table, s.lens, out, scratch, mass=mass)
    gpu_ctx.synchronize()
    m0 = mass.cpu().numpy()
    s.cache.evict(s.table, s.lens, s.lens, mass, spos, mass, spos, keep, es)
    s.cache.attention(q, s.table, s.lens, out, scratch)
    gpu_ctx.synchronize()
    for b, n in enumerate(lens):
        for h in range(hkv):
            src = torch.from_numpy(keep_of(m0[b, h, :n], np.arange(n), 1 << 40, keep)).to(DEV)
            k, v = (t[src] for t in kv[b, h])
            qq = q[b].view(hq, hd)[4 * h:4 * h + 4].double()
            ref = torch.softmax(qq @ k.T / math.sqrt(hd), -1) @ v
            assert far(out[b].view(hq, hd)[4 * h:4 * h + 4], ref, 5) <= TOL_OUT


# ---- refusals -------------------------------------------------------------------------------


def status(fn, *a, **k):
    with pytest.raises(kq.KqError) as e:
        fn(*a, **k)
    return e.value.status


def test_pools_and_sizes_that_are_refused(gpu_ctx):
    z = lambda *s: torch.zeros(s, dtype=torch.float16, device=DEV)  # noqa: E731
    assert status(paged.PagedCache, gpu_ctx, z(2, 1, 16, 96), z(2, 1, 16, 96)) == kq.KQ_ERR_UNSUPPORTED
    assert status(paged.PagedCache, gpu_ctx, z(2, 1, 24, 64), z(2, 1, 24, 64)) == kq.KQ_ERR_UNSUPPORTED
    assert status(paged.PagedCache, gpu_ctx, z(2, 1, 1040, 64), z(2, 1, 1040, 64)) == kq.KQ_ERR_UNSUPPORTED
    odd = z(3 * 16 * 64 + 8)[1:1 + 2 * 16 * 64].view(2, 1, 16, 64)
    assert status(paged.PagedCache, gpu_ctx, odd, odd) == kq.KQ_ERR_INVALID_ARG
    c = paged.PagedCache(gpu_ctx, z(4, 2, 16, 64), z(4, 2, 16, 64))
    bad = kq.KQ_ERR_INVALID_ARG
    assert status(c.scratch, 0, 2) == bad and status(c.scratch, 1, 3) == bad and status(c.scratch, 1, 34) == bad
    f, i = dict(device=DEV), dict(dtype=torch.int32, device=DEV)
    table, lens, q, out = torch.zeros((1, 2), **i), torch.ones(1, **i), torch.zeros((1, 128), **f), torch.zeros((1, 128), **f)
    scratch = c.scratch(1, 2)
    assert status(c.attention, q, table, lens, out, scratch[256:]) == kq.KQ_ERR_SHORT_BUFFER
    assert status(c.attention, q, table, lens, out, torch.zeros(scratch.numel() + 256, dtype=torch.uint8, **f)[8:]) == bad
    assert status(c.attention, q.half(), table, lens, out, scratch) == bad
    assert status(c.attention, q, table.long(), lens, out, scratch) == bad
    assert status(c.attention, q, table, lens.cpu(), out, scratch) == bad
    assert status(c.attention, q, table, torch.ones(2, **i), out, scratch) == bad
    assert status(c.attention, q, table, lens, out[:, :127], scratch) == bad
    assert status(c.attention, torch.zeros((1, 34 * 64), **f), table, lens, torch.zeros((1, 34 * 64), **f),
                  scratch) == kq.KQ_ERR_UNSUPPORTED  # 17 query heads per kv head
    assert status(c.attention, q, table, lens, out, scratch, mass=torch.zeros((1, 2, 9), **f)) == kq.KQ_ERR_SHORT_BUFFER
    qkv = torch.zeros((1, 6 * 64), **f)
    for theta in (0.0, -1.0, float("nan"), float("inf")):
        assert status(c.rope_attention, qkv, table, lens, out, scratch, theta=theta) == bad
        assert status(c.append, qkv, table, lens, theta=theta) == bad
    assert status(c.append, torch.zeros((2, 6 * 64), **f), table, torch.zeros(2, **i), theta=1e4) == bad
    two = torch.zeros((2, 6 * 64), **f)  # q_out over qkv at another stride
    assert status(c.append, two, table, torch.zeros(2, **i), theta=1e4, seqs=torch.zeros(2, **i),
                  q_out=two.as_strided((2, 128), (128, 1))) == bad
    m, p = torch.zeros((1, 2, 32), **f), torch.zeros((1, 2, 32), **i)
    es = c.evict_scratch(1, 32)
    assert status(c.evict, table, lens, lens, m, p, m, p, 0, es) == bad
    assert status(c.evict, table, lens, lens, m, p, m, p, 4, es[:64]) == kq.KQ_ERR_SHORT_BUFFER
    assert status(c.evict, table, lens, lens, m, p, m[:, :, :31], p, 4, es) == bad
    before = gpu_ctx.launch_count
    c.append(torch.zeros((0, 6 * 64), **f), table, torch.zeros(0, **i), theta=1e4, seqs=torch.zeros(0, **i))
    assert gpu_ctx.launch_count == before  # no rows: nothing is queued


def test_a_length_past_the_table_leaves_the_cache_alone(gpu_ctx):
    """A sequence that outgrew its table is an idle row: its last slot is not overwritten,
    evicting it changes neither its length nor its rows."""
    hd, hkv, page = 64, 2, 16
    s = Setup(gpu_ctx, [48, 20], 2, hkv, hd, page, seed=2)
    table = s.table[:, :3].clamp(0, s.pages - 1).contiguous()
    lens = torch.tensor([49, 21], dtype=torch.int32, device=DEV)
    qkv, out = torch.randn((2, 6 * hd), device=DEV), torch.full((2, 2 * hd), 7.0, device=DEV)
    m, p = torch.rand((2, hkv, 48), device=DEV), torch.arange(48, dtype=torch.int32, device=DEV).expand(2, hkv, 48).contiguous()
    scratch, es = s.cache.scratch(2, 2, 48), s.cache.evict_scratch(2, 48)
    rows = [s.k[s.table[0, j // page].long(), :, j % page].clone() for j in range(48)]
    m0, p0 = m.clone(), p.clone()
    torch.cuda.synchronize()
    s.cache.rope_attention(qkv, table, lens, out, scratch, theta=1e4, mass=m, slot_pos=p)
    assert status(gpu_ctx.synchronize) == kq.KQ_ERR_INVALID_ARG
    s.cache.evict(table, lens, lens, m, p, m, p, 30, es)
    assert status(gpu_ctx.synchronize) == kq.KQ_ERR_INVALID_ARG
    assert lens.tolist() == [49, 21]
    assert torch.equal(out[0], torch.zeros_like(out[0])) and out[1].isfinite().all() and bool(out[1].abs().max() > 0)
    assert torch.equal(m[0], m0[0]) and torch.equal(p[0], p0[0])
    for j in range(48):
        assert torch.equal(s.k[s.table[0, j // page].long(), :, j % page], rows[j])


@pytest.mark.parametrize("what", ["page", "negative", "far page", "len", "negative len", "slot", "far slot", "seq"])
def test_what_lies_outside_is_reported_and_not_followed(gpu_ctx, what):
    hd, hkv, page = 64, 2, 16
    s = Setup(gpu_ctx, [40, 20], 2, hkv, hd, page, seed=1)
    table, lens = s.table.clone(), s.lens.clone()
    if what in ("page", "negative", "far page"):
        table[0, 1] = {"page": s.pages, "negative": -1, "far page": 2 ** 31 - 1}[what]
    if what in ("len", "negative len"):
        lens[0] = {"len": table.shape[1] * page + 1, "negative len": -3}[what]
        table.clamp_(0, s.pages - 1)
    q, out = torch.randn((2, 2 * hd), device=DEV), torch.zeros((2, 2 * hd), device=DEV)
    m, p = torch.rand((2, hkv, 48), device=DEV), torch.zeros((2, hkv, 48), dtype=torch.int32, device=DEV)
    scratch, es = s.cache.scratch(2, 2, 48), s.cache.evict_scratch(2, 48)
    k0 = s.k.clone()
    torch.cuda.synchronize()
    if what in ("slot", "far slot", "seq"):
        qkv = torch.randn((2, 6 * hd), device=DEV)
        slots = torch.tensor([{"slot": 48, "far slot": -2, "seq": 3}[what], -1], dtype=torch.int32, device=DEV)
        seqs = torch.tensor([2 if what == "seq" else 0, 0], dtype=torch.int32, device=DEV)
        table = table[:, :3].contiguous()
        torch.cuda.synchronize()
        s.cache.append(qkv, table, slots, theta=1e4, seqs=seqs)
        assert status(gpu_ctx.synchronize) == kq.KQ_ERR_INVALID_ARG
        assert torch.equal(s.k.nan_to_num(7), k0.nan_to_num(7))
        return
    s.cache.attention(q, table, lens, out, scratch)
    assert status(gpu_ctx.synchronize) == kq.KQ_ERR_INVALID_ARG
    lens2, m2, p2 = lens.clone(), m.clone(), p.clone()
    torch.cuda.synchronize()
    s.cache.evict(table, lens, lens2, m, p, m2, p2, 10, es)
    assert status(gpu_ctx.synchronize) == kq.KQ_ERR_INVALID_ARG
    # the other sequence and the context are fine
    s.cache.attention(q, s.table, s.lens, out, scratch)
    gpu_ctx.synchronize()
