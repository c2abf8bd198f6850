"""Calls of the paged cache as a server mixes them on one context: what one call
leaves behind for the next, block tables cut out of wider ones, infinite keys,
and what the calls do with the sequences that are in order beside one that is
not.  Definitions and tolerances are those of test_gpu_paged."""
import math

import numpy as np
import pytest
import torch

from pesti_b200 import decoder as dec
from pesti_b200 import kq, paged, synthetic
from test_gpu_paged import DEV, TOL_OUT, Setup, far, keep_of, status, turn
from test_gpu_serving import LLAMA_TINY

pytestmark = pytest.mark.gpu


# ---- input out of bounds and the calls behind it ---------------------------------------------


def test_bad_input_leaves_the_other_calls_on_the_context_alone(gpu_ctx):
    """A row past its table, then a whole decode step in one kernel (its grid barriers and
    exchange words are waited for) and a synchronous linear, before anything is synchronized:
    both as without the row, which the context's own synchronize reports, once."""
    model = dec.Decoder(LLAMA_TINY, gpu_ctx, 1, 20, max_new=4, seed=5, step_kernel=True)
    assert model.step_kernel
    s = Setup(gpu_ctx, [40], 2, 2, 64, 16, seed=71)
    table = s.table[:, :3].contiguous()
    qkv = torch.randn((1, 6 * 64), generator=s.g, device=DEV)
    slots = torch.tensor([48], dtype=torch.int32, device=DEV)
    raw = synthetic.gguf_weight(kq.KQ_GGUF_Q4_K, 512, 1024, seed=1)
    w = kq.Weight(gpu_ctx, kq.KQ_GGUF_Q4_K, raw, 512, 1024)
    x, y, y2 = torch.randn((1, 1024), generator=s.g, device=DEV), torch.zeros(512, device=DEV), torch.zeros(512, device=DEV)
    model.tokens.fill_(7)
    torch.cuda.synchronize()
    model.step(20)
    w.linear(x, 1, y, device_ptrs=True, sync=True)
    gpu_ctx.synchronize()
    want = model.logits.clone()
    for _ in range(20):
        model.logits.fill_(9.0)
        torch.cuda.synchronize()
        s.cache.append(qkv, table, slots, theta=1e4)
        for _ in range(4):  # the same step again: it writes the same row of its cache
            model.step(20)
        w.linear(x, 1, y2, device_ptrs=True, sync=True)
        torch.cuda.synchronize()
        assert torch.equal(model.logits, want) and torch.equal(y2, y)
        assert status(gpu_ctx.synchronize) == kq.KQ_ERR_INVALID_ARG
        gpu_ctx.synchronize()
    w.free()
    model.close()


# ---- appended keys ------------------------------------------------------------------------


@pytest.mark.parametrize("hd,hkv", [(64, 1), (64, 4), (128, 8), (256, 2)])
def test_append_stores_the_exact_key_rounded(gpu_ctx, hd, hkv):
    """As for a step's key: turned in 64 bits, to the nearest f32, to the nearest f16.  The
    first rounding moves the second at about 1e-7 of the elements; sums in f32 would move 2e-4 of
    them, some fifty of these 262,144."""
    n, hq, theta = 262144 // (hd * hkv), hkv, 1e6
    s = Setup(gpu_ctx, [n], hq, hkv, hd, 16, seed=hd)
    qkv = torch.randn((n, (hq + 2 * hkv) * hd), generator=s.g, device=DEV)
    pos = torch.randint(0, 120000, (n,), generator=s.g, device=DEV).int()
    slots, seqs = torch.arange(n, dtype=torch.int32, device=DEV), torch.zeros(n, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    s.cache.append(qkv, s.table, slots, theta=theta, seqs=seqs, pos=pos)
    gpu_ctx.synchronize()
    want = turn(qkv.view(n, hq + 2 * hkv, hd)[:, hq:hq + hkv], pos, theta).half()
    at = s.table[0, slots.long() // 16].long()
    assert int((s.k[at, :, slots.long() % 16] != want).sum()) <= 2


@pytest.mark.parametrize("hd,hq,hkv", [(64, 14, 2), (128, 32, 8), (256, 9, 1)])
def test_append_and_a_step_store_the_same_keys(gpu_ctx, hd, hq, hkv):
    """A token that is appended again later finds the bits that its own step wrote."""
    B, theta = 400, 5e5
    s = Setup(gpu_ctx, [3] * B, hq, hkv, hd, 16, seed=hd + 1)
    qkv = 3.0 * torch.randn((B, (hq + 2 * hkv) * hd), generator=s.g, device=DEV)
    pos = torch.randint(0, 1 << 20, (B,), generator=s.g, device=DEV).int()
    out = torch.zeros((B, hq * hd), device=DEV)
    again = paged.PagedCache(gpu_ctx, s.k.clone(), s.v.clone())
    scratch = s.cache.scratch(B, hq)
    torch.cuda.synchronize()
    s.cache.rope_attention(qkv, s.table, s.lens, out, scratch, theta=theta, pos=pos)
    again.append(qkv, s.table, s.lens - 1, theta=theta, pos=pos)
    gpu_ctx.synchronize()
    at = s.table[:, 0].long()
    assert torch.equal(s.k[at, :, 2], again.k[at, :, 2]) and torch.equal(s.v[at, :, 2], again.v[at, :, 2])


# ---- weights of slots that are used again ----------------------------------------------------


def test_appended_slots_start_without_weight(gpu_ctx):
    """Evict, append a chunk into the freed slots, attend, evict: the new slots are ranked by the
    weights they gathered themselves, not by those of the tokens that lay there."""
    hd, hq, hkv, page, lens, keep, more = 64, 4, 2, 16, [60, 45], 20, 12
    s = Setup(gpu_ctx, lens, hq, hkv, hd, page, seed=21)
    B, ld = 2, 64
    spos = torch.arange(ld, dtype=torch.int32, device=DEV).expand(B, hkv, ld).contiguous()
    mass = torch.rand((B, hkv, ld), generator=s.g, device=DEV)
    mass[:, :, keep:] += 100.0  # cut off, these weights stay behind in the array
    mass[:, :, :keep] += 200.0
    chunk = torch.randn((B * more, (hq + 2 * hkv) * hd), generator=s.g, device=DEV)
    q = torch.randn((B, hq * hd), generator=s.g, device=DEV)
    seqs = torch.arange(B, dtype=torch.int32, device=DEV).repeat_interleave(more)
    slots = (keep + torch.arange(more, dtype=torch.int32, device=DEV)).repeat(B)
    slots[more - 1] = -1  # a row that is left out
    grown = torch.tensor([keep + more - 1, keep + more], dtype=torch.int32, device=DEV)
    out, scratch, es = torch.empty_like(q), s.cache.scratch(B, hq, ld), s.cache.evict_scratch(B, ld)
    torch.cuda.synchronize()
    s.cache.evict(s.table, s.lens, s.lens, mass, spos, mass, spos, keep, es)
    gpu_ctx.synchronize()
    old = mass.clone()
    s.cache.append(chunk, s.table, slots, theta=1e4, seqs=seqs, pos=slots + 100, mass=mass, slot_pos=spos)
    gpu_ctx.synchronize()
    want = old.clone()
    for b, n in enumerate(grown.tolist()):
        want[b, :, keep:n] = 0.0
    assert torch.equal(mass, want)
    assert (spos[1, :, keep:keep + more] == slots[more:] + 100).all() and (spos[0, :, keep + more - 1] < 100).all()
    s.lens_h, s.lens = grown.tolist(), grown
    torch.cuda.synchronize()
    s.cache.attention(q, s.table, s.lens, out, scratch, mass=mass)
    gpu_ctx.synchronize()
    _, ref = s.reference(q.view(B, hq, hd))
    for (b, h), m in ref.items():
        # the weight's own bound, and half a step of f32 of a sum near 200
        assert float((mass[b, h, :len(m)] - want[b, h, :len(m)] - m).abs().max()) <= TOL_OUT * 2 + 2 ** -16
    m0 = mass.cpu().numpy()
    s.cache.evict(s.table, s.lens, s.lens, mass, spos, mass, spos, keep + 5, es)
    gpu_ctx.synchronize()
    for b, n in enumerate([keep + more - 1, keep + more]):
        for h in range(hkv):
            src = keep_of(m0[b, h, :n], np.arange(n), 1 << 40, keep + 5)
            assert np.array_equal(src[:keep], np.arange(keep))  # the old slots, at 200 and more
            assert np.array_equal(mass[b, h, :keep + 5].cpu().numpy(), m0[b, h, src])


def test_append_checks_the_tracked_slots(gpu_ctx):
    """mass alone, slot_pos alone, and slots past what is tracked."""
    hd, hkv = 64, 2
    s = Setup(gpu_ctx, [40, 30], 2, hkv, hd, 16, seed=22)
    qkv = torch.randn((2, 6 * hd), generator=s.g, device=DEV)
    slots = torch.tensor([39, 7], dtype=torch.int32, device=DEV)
    mass = torch.ones((2, hkv, 40), device=DEV)
    torch.cuda.synchronize()
    s.cache.append(qkv, s.table, slots, theta=1e4, mass=mass)
    gpu_ctx.synchronize()
    want = torch.ones_like(mass)
    want[0, :, 39] = want[1, :, 7] = 0.0
    assert torch.equal(mass, want)
    short = torch.ones((2, hkv, 39), device=DEV)
    k0 = s.k.clone()
    torch.cuda.synchronize()
    s.cache.append(3 * qkv, s.table, slots, theta=1e4, mass=short)
    assert status(gpu_ctx.synchronize) == kq.KQ_ERR_INVALID_ARG  # slot 39 of 39: that row is left out
    assert (short[0] == 1).all() and (short[1, :, 7] == 0).all() and int((short == 0).sum()) == hkv
    at = int(s.table[0, 2])
    assert torch.equal(s.k[at].nan_to_num(7), k0[at].nan_to_num(7))
    bad = kq.KQ_ERR_INVALID_ARG
    spos = torch.zeros((2, hkv, 41), dtype=torch.int32, device=DEV)
    assert status(s.cache.append, qkv, s.table, slots, theta=1e4, mass=mass, slot_pos=spos) == bad
    assert status(s.cache.append, qkv, s.table, slots, theta=1e4, mass=mass.double()) == bad
    assert status(s.cache.append, qkv, s.table, slots, theta=1e4, mass=mass[:1]) == bad


# ---- block tables cut out of wider ones -------------------------------------------------------


@pytest.mark.parametrize("first", [0, 2])
def test_a_narrowed_table_bounds_lengths_and_slots_by_its_own_width(gpu_ctx, first):
    """Three columns of a table of ten whose other entries name pages that hold other rows."""
    hd, hq, hkv, page, cols = 64, 4, 2, 16, 3
    full = cols * page
    s = Setup(gpu_ctx, [full, 20, full], hq, hkv, hd, page, seed=31, spare=4)
    s.k.nan_to_num_(3.0)
    s.v.nan_to_num_(3.0)
    named = torch.zeros(s.pages, dtype=torch.bool)
    for b, n in enumerate(s.lens_h):
        named[s.table[b, :-(-n // page)].long().cpu()] = True
    spare = torch.nonzero(~named)[0].int().to(DEV)
    wide = spare.repeat(3, 10)
    wide[:, first:first + cols] = s.table[:, :cols].clamp(0, s.pages - 1)
    wide[1, first + 2:first + cols] = spare
    table = wide[:, first:first + cols]
    assert not table.is_contiguous()
    qkv = torch.randn((3, (hq + 2 * hkv) * hd), generator=s.g, device=DEV)
    q = qkv[:, :hq * hd].contiguous()
    out = torch.full((3, hq * hd), 7.0, device=DEV)
    ld = 10 * page
    mass, spos = torch.rand((3, hkv, ld), generator=s.g, device=DEV), torch.zeros((3, hkv, ld), dtype=torch.int32, device=DEV)
    scratch, es = s.cache.scratch(3, hq, ld), s.cache.evict_scratch(3, ld)
    lens = torch.tensor([full + 1, 20, full], dtype=torch.int32, device=DEV)
    k0, v0, m0 = s.k.clone(), s.v.clone(), mass.clone()
    torch.cuda.synchronize()

    s.cache.attention(q, table, lens, out, scratch)
    assert status(gpu_ctx.synchronize) == kq.KQ_ERR_INVALID_ARG
    s.lens_h = [0, 20, full]
    ref, _ = s.reference(q.view(3, hq, hd))
    assert far(out.view(3, hq, hd), ref, float(s.v.abs().max())) <= TOL_OUT
    assert not out[0].any()

    slots, seqs = torch.tensor([full, 5], dtype=torch.int32, device=DEV), torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    s.cache.append(qkv[:2], table, slots, theta=1e4, seqs=seqs)
    assert status(gpu_ctx.synchronize) == kq.KQ_ERR_INVALID_ARG
    at = int(table[1, 0])
    k0[at, :, 5], v0[at, :, 5] = s.k[at, :, 5], s.v[at, :, 5]
    assert torch.equal(s.k, k0) and torch.equal(s.v, v0)
    assert torch.equal(v0[at, :, 5], qkv[1].view(-1, hd)[hq + hkv:].half())

    s.cache.rope_attention(qkv, table, lens, out, scratch, theta=1e4, mass=mass, slot_pos=spos)
    assert status(gpu_ctx.synchronize) == kq.KQ_ERR_INVALID_ARG
    for b, n in ((1, 20), (2, full)):
        at, r = int(table[b, (n - 1) // page]), (n - 1) % page
        k0[at, :, r], v0[at, :, r] = s.k[at, :, r], s.v[at, :, r]
        assert torch.equal(v0[at, :, r], qkv[b].view(-1, hd)[hq + hkv:].half())
    assert torch.equal(s.k, k0) and torch.equal(s.v, v0)
    assert not out[0].any() and torch.equal(mass[0], m0[0])

    lens2, m2, p2 = torch.zeros_like(lens), mass.clone(), spos.clone()
    torch.cuda.synchronize()
    s.cache.evict(table, lens, lens2, mass, spos, m2, p2, 10, es)
    assert status(gpu_ctx.synchronize) == kq.KQ_ERR_INVALID_ARG
    assert lens2.tolist() == [full + 1, 10, 10]
    ids = table[0].long()
    assert torch.equal(s.k[ids], k0[ids]) and torch.equal(s.k[spare.long()], k0[spare.long()])

    # the next call takes the width of its own table again
    s.lens_h = [20, 1]
    two = torch.tensor(s.lens_h, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    s.cache.attention(q[:2], s.table[:2], two, out[:2], scratch)
    gpu_ctx.synchronize()
    assert far(out[:2].view(2, hq, hd), s.reference(q[:2].view(2, hq, hd))[0], float(s.v.abs().max())) <= TOL_OUT


def test_a_narrowed_table_is_captured_with_its_width(gpu_ctx):
    """Two graphs over one handle, one with the whole table and one with a part of it."""
    hd, hq, hkv, page = 64, 2, 2, 16
    s = Setup(gpu_ctx, [70, 30], hq, hkv, hd, page, seed=32)
    part = s.table[:, :2]
    q = torch.randn((2, hq * hd), generator=s.g, device=DEV)
    outs = [torch.empty_like(q) for _ in range(2)]
    scratch = s.cache.scratch(2, hq)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    gpu_ctx.set_stream(stream)
    try:
        s.cache.attention(q, s.table, s.lens, outs[0], scratch)
        gpu_ctx.synchronize()
        graphs = []
        for table, out in zip((s.table, part), outs):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                s.cache.attention(q, table, s.lens, out, scratch)
            graphs.append(g)
        ref, _ = s.reference(q.view(2, hq, hd))
        for k in (0, 1, 0):
            outs[k].fill_(9.0)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                graphs[k].replay()
            if k:
                assert status(gpu_ctx.synchronize) == kq.KQ_ERR_INVALID_ARG
            else:
                gpu_ctx.synchronize()
            want = ref.clone()
            if k:
                want[0] = 0.0  # 70 slots do not fit two pages of 16
            assert far(outs[k].view(2, hq, hd), want, 5) <= TOL_OUT
        del graphs, g
    finally:
        gpu_ctx.set_stream(None)


# ---- infinite keys ------------------------------------------------------------------------------


@pytest.mark.parametrize("hd,hq,hkv,page", [(64, 14, 2, 16), (128, 32, 8, 64), (256, 9, 1, 48)])
def test_infinite_keys_weigh_nothing_or_are_reported_as_nan(gpu_ctx, hd, hq, hkv, page):
    """A score of -inf takes its slot out; one of +inf, or scores that are all -inf, leave no
    softmax: NaN, in the rows of that sequence and head alone."""
    lens = [200, 64, 5000, 16, 70, 3]
    s = Setup(gpu_ctx, lens, hq, hkv, hd, page, seed=hd)
    B, G = len(lens), hq // hkv
    q = torch.randn((B, hkv, G, hd), generator=s.g, device=DEV)
    q[:, :, :, 3], q[:, :, :, hd - 1] = q[:, :, :, 3].abs() + 0.1, -q[:, :, :, hd - 1].abs() - 0.1
    q = q.reshape(B, hq * hd).contiguous()

    def put(b, slots, d, x, head=slice(None)):
        for j in slots:
            s.k[int(s.table[b, j // page]), head, j % page, d] = x

    inf = float("inf")
    put(0, [0, 5, 40, 199], 3, -inf)                 # single slots
    put(0, [77], hd - 1, inf)
    put(0, [78], 3, -inf)                            # two infinities of one slot that agree
    put(0, [78], hd - 1, inf)
    put(1, range(16, 32), 3, -inf)                   # all 16 slots of a warp
    put(2, range(0, 3000), 3, -inf)                  # the first tiles of a sequence that CTAs share
    put(3, range(1, 16), 3, -inf)                    # all slots but one
    put(4, [7], 3, inf, 0)                           # +inf, in one kv head
    put(5, range(3), 3, -inf, hkv - 1)               # nothing left, in one kv head
    ld = max(lens)
    out, mass = torch.empty_like(q), torch.zeros((B, hkv, ld), device=DEV)
    scratch = s.cache.scratch(B, hq, ld)
    torch.cuda.synchronize()
    s.cache.attention(q, s.table, s.lens, out, scratch, mass=mass)
    gpu_ctx.synchronize()
    ref, ref_mass = s.reference(q.view(B, hq, hd))
    got = out.view(B, hq, hd)
    assert torch.equal(got.isnan(), ref.isnan())
    assert ref[4, :G].isnan().all() and ref[5, hq - G:].isnan().all() and int(ref.isnan().sum()) == 2 * G * hd
    vmax = float(s.v.nan_to_num(0).abs().max())
    assert far(got.nan_to_num(0), ref.nan_to_num(0), vmax) <= TOL_OUT
    for (b, h), m in ref_mass.items():
        assert torch.equal(mass[b, h, :len(m)].isnan(), m.isnan())
        assert float((mass[b, h, :len(m)].nan_to_num(0) - m.nan_to_num(0)).abs().max()) <= TOL_OUT * G
    plain = torch.empty_like(q)  # without the weights: the same output
    s.cache.attention(q, s.table, s.lens, plain, scratch)
    gpu_ctx.synchronize()
    assert torch.equal(plain.nan_to_num(9), out.nan_to_num(9))


def test_a_key_past_the_range_of_f16_is_stored_as_infinite(gpu_ctx):
    """It takes its slot out, or leaves NaN, as its sign says; the other heads are not touched."""
    hd, hq, hkv = 64, 2, 2
    s = Setup(gpu_ctx, [40], hq, hkv, hd, 16, seed=41)
    qkv = torch.randn((1, 6 * hd), generator=s.g, device=DEV)
    qkv[0, 9], qkv[0, 2 * hd + 9] = 2.0, -1e6
    pos, lens = torch.zeros(1, dtype=torch.int32, device=DEV), s.lens
    out, scratch = torch.empty((1, hq * hd), device=DEV), s.cache.scratch(1, hq)
    torch.cuda.synchronize()
    s.cache.rope_attention(qkv, s.table, lens, out, scratch, theta=1e4, pos=pos)
    gpu_ctx.synchronize()
    assert float(s.k[int(s.table[0, 2]), 0, 39 - 32, 9]) == -math.inf
    ref, _ = s.reference(qkv[:, :hq * hd].view(1, hq, hd))  # position 0 turns nothing
    assert torch.isfinite(ref).all()
    assert far(out.view(1, hq, hd), ref, float(s.v.nan_to_num(0).abs().max())) <= TOL_OUT


# ---- budgets past 32 bits ------------------------------------------------------------------------


@pytest.mark.parametrize("keep", [2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, 2 ** 63 + 1])
def test_a_budget_past_32_bits_keeps_everything(gpu_ctx, keep):
    s = Setup(gpu_ctx, [30, 7], 2, 2, 64, 16, seed=51)
    m, p = torch.rand((2, 2, 30), device=DEV), torch.arange(30, dtype=torch.int32, device=DEV).expand(2, 2, 30).contiguous()
    es, lens, k0 = s.cache.evict_scratch(2, 30), torch.zeros_like(s.lens), s.k.clone()
    m0 = m.clone()
    torch.cuda.synchronize()
    s.cache.evict(s.table, s.lens, lens, m, p, m, p, keep, es)
    gpu_ctx.synchronize()
    assert lens.tolist() == [30, 7]
    assert torch.equal(m, m0) and torch.equal(s.k.nan_to_num(7), k0.nan_to_num(7))


# ---- sizes ----------------------------------------------------------------------------------------


def test_scratch_sizes_past_64_bits_are_refused(gpu_ctx):
    """Not a small remainder of them (sizes only: nothing is queued)."""
    pool = torch.zeros((1, 32768, 16, 64), dtype=torch.float16, device=DEV)
    cache = paged.PagedCache(gpu_ctx, pool, pool.clone())
    most = 2 ** 31 - 1
    bad = kq.KQ_ERR_INVALID_ARG
    # 65535 x 32768 pairs of 2^31 slots: 2^65 bytes of scores, 2^64 of lists
    assert status(cache.scratch, 65535, 32768, most) == bad
    assert status(cache.evict_scratch, 65535, most) == bad
    n = cache.lib.kq_kv_evict_scratch(cache.handle, 4096, 1 << 20)
    assert n == 4096 * 32768 * (16 + 4 * (1 << 20))
    n = cache.lib.kq_kv_attention_scratch(cache.handle, 64, 32768, 1 << 20)
    assert n > 64 * 32768 * 2 * 4 * (1 << 20)


def test_a_paged_decoder_holds_no_scratch_of_the_contiguous_attention(gpu_ctx):
    model = dec.Decoder(LLAMA_TINY, gpu_ctx, 2, 20, max_new=4, seed=5, page_size=16)
    plain = dec.Decoder(LLAMA_TINY, gpu_ctx, 2, 20, max_new=4, seed=5)
    model.tokens.copy_(torch.tensor([3, 4], dtype=torch.int32))
    torch.cuda.synchronize()
    model.step()
    gpu_ctx.synchronize()
    assert torch.isfinite(model.logits).all() and bool(model.logits.abs().max() > 0)
    assert hasattr(plain, "att_scratch") and not hasattr(model, "att_scratch")
    model.close()
    plain.close()


# ---- the sequences beside one that is out of bounds ------------------------------------------------


@pytest.mark.parametrize("what", ["page", "negative", "far page", "len", "negative len"])
def test_the_other_sequences_are_right_beside_one_out_of_bounds(gpu_ctx, what):
    """Attention and eviction give them what they give alone, and nothing outside the pages of
    the sequences is written."""
    hd, hq, hkv, page, keep = 64, 4, 2, 16, 10
    s = Setup(gpu_ctx, [40, 20, 33], hq, hkv, hd, page, seed=61)
    table, lens = s.table.clone(), s.lens.clone()
    long = what in ("len", "negative len")
    if long:
        lens[0] = {"len": table.shape[1] * page + 1, "negative len": -3}[what]
    else:
        table[0, 1] = {"page": s.pages, "negative": -1, "far page": 2 ** 31 - 1}[what]
    q, out = torch.randn((3, hq * hd), generator=s.g, device=DEV), torch.full((3, hq * hd), 7.0, device=DEV)
    m, p = torch.rand((3, hkv, 48), generator=s.g, device=DEV), torch.zeros((3, hkv, 48), dtype=torch.int32, device=DEV)
    p += torch.arange(48, dtype=torch.int32, device=DEV)
    scratch, es = s.cache.scratch(3, hq, 48), s.cache.evict_scratch(3, 48)
    ref, _ = s.reference(q.view(3, hq, hd))
    k0, v0, m0, p0 = s.k.clone(), s.v.clone(), m.cpu().numpy(), p.cpu().numpy()
    old = {(b, h): (s.rows(s.k, b, h, n), s.rows(s.v, b, h, n)) for b, n in enumerate(s.lens_h) for h in range(hkv)}
    vmax = float(s.v.nan_to_num(0).abs().max())
    torch.cuda.synchronize()
    s.cache.attention(q, table, lens, out, scratch)
    assert status(gpu_ctx.synchronize) == kq.KQ_ERR_INVALID_ARG
    gpu_ctx.synchronize()  # reported once
    assert far(out[1:].view(2, hq, hd), ref[1:], vmax) <= TOL_OUT
    if long:
        assert not out[0].any()
    assert torch.equal(s.k.nan_to_num(7), k0.nan_to_num(7)) and torch.equal(s.v.nan_to_num(7), v0.nan_to_num(7))

    lens2, m2, p2 = torch.full_like(lens, -9), torch.full_like(m, 77.0), torch.full_like(p, -77)
    torch.cuda.synchronize()
    s.cache.evict(table, lens, lens2, m, p, m2, p2, keep, es)
    assert status(gpu_ctx.synchronize) == kq.KQ_ERR_INVALID_ARG
    assert lens2.tolist() == [int(lens[0]) if long else keep, keep, keep]
    assert np.array_equal(m.cpu().numpy(), m0) and np.array_equal(p.cpu().numpy(), p0)
    if long:
        assert (m2[0] == 77).all() and (p2[0] == -77).all()
    mine = torch.zeros(s.pages, dtype=torch.bool, device=DEV)
    for b in (1, 2) if long else (0, 1, 2):
        ids = table[b, :-(-s.lens_h[b] // page)].long()
        mine[ids[(ids >= 0) & (ids < s.pages)]] = True
    for pool, before in ((s.k, k0), (s.v, v0)):
        assert torch.equal(pool[~mine].nan_to_num(7), before[~mine].nan_to_num(7))
    for b in (1, 2):
        for h in range(hkv):
            src = keep_of(m0[b, h, :s.lens_h[b]], p0[b, h, :s.lens_h[b]], 1 << 40, keep)
            assert np.array_equal(m2[b, h, :keep].cpu().numpy(), m0[b, h, src])
            assert np.array_equal(p2[b, h, :keep].cpu().numpy(), p0[b, h, src])
            assert (m2[b, h, keep:] == 77).all() and (p2[b, h, keep:] == -77).all()
            for pool, rows in zip((s.k, s.v), old[b, h]):
                assert torch.equal(s.rows(pool, b, h, keep), rows[torch.from_numpy(src).to(DEV)])

    # and the next valid call is right for every sequence
    for pool, before in ((s.k, k0), (s.v, v0)):
        pool.copy_(before)
    torch.cuda.synchronize()
    s.cache.attention(q, s.table, s.lens, out, scratch)
    gpu_ctx.synchronize()
    assert far(out.view(3, hq, hd), ref, vmax) <= TOL_OUT


@pytest.mark.parametrize("what", ["slot", "far slot", "seq", "negative seq", "page"])
def test_the_other_rows_are_appended_beside_one_out_of_bounds(gpu_ctx, what):
    hd, hq, hkv, page = 64, 2, 2, 16
    s = Setup(gpu_ctx, [40, 20], hq, hkv, hd, page, seed=62)
    table = s.table[:, :3].contiguous()
    qkv = torch.randn((3, 6 * hd), generator=s.g, device=DEV)
    slots = torch.tensor([5, {"slot": 48, "far slot": -2, "page": 17}.get(what, 0), 19], dtype=torch.int32, device=DEV)
    seqs = torch.tensor([0, {"seq": 2, "negative seq": -1}.get(what, 0), 1], dtype=torch.int32, device=DEV)
    if what == "page":
        table[0, 1] = s.pages
    k0, v0 = s.k.clone(), s.v.clone()
    torch.cuda.synchronize()
    s.cache.append(qkv, table, slots, theta=1e4, seqs=seqs)
    assert status(gpu_ctx.synchronize) == kq.KQ_ERR_INVALID_ARG
    rows = qkv.view(3, 3 * hkv, hd)
    want = turn(rows[:, hq:hq + hkv], slots, 1e4).half()
    for i, (b, t) in ((0, (0, 5)), (2, (1, 19))):
        at = int(s.table[b, t // page])
        k0[at, :, t % page], v0[at, :, t % page] = want[i], rows[i, hq + hkv:].half()
    assert torch.equal(s.v.nan_to_num(7), v0.nan_to_num(7))
    # the two roundings of a key differ from one at 1e-7 of the elements
    assert int((s.k.nan_to_num(7) != k0.nan_to_num(7)).sum()) <= 1


# ---- far positions -----------------------------------------------------------------------------


@pytest.mark.parametrize("hd,hq,hkv", [(64, 14, 2), (128, 32, 8), (256, 9, 1)])
def test_rotated_attention_is_as_exact_at_far_positions(gpu_ctx, hd, hq, hkv):
    """A turned q element is off by four roundings (scale, cosine and sine, a product, the sum) of
    its pair's length, sqrt(2) of the element on average: 5.7 x 2^-24 of it.  With sum |q_i k_i| /
    sqrt(hd) about 11 at 128 and 15 at 256, a score by 15 x 3.4e-7 = 5.1e-6 more than the 1.1e-5 of
    a given q, an output by twice the sum: 3.2e-5, and a quarter on top for the largest of the
    rows.  An f32 angle would be off by 4e-3 here."""
    lens = [40, 700, 1, 2049, 130]
    s = Setup(gpu_ctx, lens, hq, hkv, hd, 16, seed=81)
    B = len(lens)
    qkv = 1.5 * torch.randn((B, (hq + 2 * hkv) * hd), generator=s.g, device=DEV)
    pos = torch.randint(90000, 131072, (B,), generator=s.g, device=DEV).int()
    out, scratch = torch.empty((B, hq * hd), device=DEV), s.cache.scratch(B, hq)
    torch.cuda.synchronize()
    s.cache.rope_attention(qkv, s.table, s.lens, out, scratch, theta=5e5, pos=pos)
    gpu_ctx.synchronize()
    q = turn(qkv.view(B, hq + 2 * hkv, hd)[:, :hq], pos, 5e5)
    ref, _ = s.reference(q)
    assert far(out.view(B, hq, hd), ref, float(s.v.nan_to_num(0).abs().max())) <= 4e-5
