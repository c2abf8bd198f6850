"""A decoder on a paged cache: the same logits as on the contiguous cache, steps of
sequences with positions of their own, sampling from the step's logits, and
eviction between steps, as a server runs them together."""
import numpy as np
import pytest
import torch

from pesti_b200 import decoder as dec

pytestmark = pytest.mark.gpu

LLAMA_TINY = dec.DecoderConfig("llama-like-tiny", 2, 512, 4, 2, 128, 768, 300, 1e-5, 5e5, False)
QWEN_TINY = dec.DecoderConfig("qwen-like-tiny", 2, 448, 7, 1, 64, 512, 300, 1e-6, 1e6, True)
# an attention output's f32 rounding, and a cached key's f16 step where the two kernels' angles
# differ, pass through two layers whose activations are quantized to 15 bits: the decoder tests' bound
TOL = 2e-3


def rel_err(y, ref):
    return float((y.double() - ref.double()).abs().max() / ref.double().abs().max())


@pytest.mark.parametrize("cfg", [LLAMA_TINY, QWEN_TINY], ids=lambda c: c.name)
@pytest.mark.parametrize("batch,page", [(1, 16), (3, 64)])
def test_paged_steps_match_contiguous_steps(gpu_ctx, cfg, batch, page):
    plain = dec.Decoder(cfg, gpu_ctx, batch, 40, max_new=4, seed=3)
    model = dec.Decoder(cfg, gpu_ctx, batch, 40, max_new=4, seed=3, page_size=page)
    for step in range(3):
        toks = torch.tensor([(7 * step + 50 * b) % cfg.vocab for b in range(batch)], dtype=torch.int32)
        for m in (plain, model):
            m.tokens.copy_(toks)
        model.lens.fill_(41 + step)
        model.positions.fill_(40 + step)
        torch.cuda.synchronize()
        plain.step(40 + step)
        model.step()
        gpu_ctx.synchronize()
        assert rel_err(model.logits, plain.logits) <= TOL
    with pytest.raises(ValueError):
        model.step(41)
    with pytest.raises(ValueError):
        plain.step()
    plain.close()
    model.close()


def test_sequences_at_positions_of_their_own(gpu_ctx):
    """A ragged batch gives each sequence what it gets in a batch of one; an idle row disturbs none."""
    cfg, ctx_len = LLAMA_TINY, 60
    model = dec.Decoder(cfg, gpu_ctx, 4, ctx_len, max_new=4, seed=5, page_size=16)
    lens = [61, 0, 1, 33]
    model.tokens.copy_(torch.tensor([5, -1, 9, 250], dtype=torch.int32))
    model.lens.copy_(torch.tensor(lens, dtype=torch.int32))
    model.positions.copy_(torch.tensor([60, 0, 0, 32], dtype=torch.int32))
    caches = [(L["k"].clone(), L["v"].clone()) for L in model.layers]
    torch.cuda.synchronize()
    model.step()
    gpu_ctx.synchronize()
    got = model.logits.clone()
    for b in (0, 2, 3):
        for L, (k, v) in zip(model.layers, caches):
            L["k"].copy_(k)
            L["v"].copy_(v)
        alone = torch.zeros(4, dtype=torch.int32)
        alone[b] = lens[b]
        model.lens.copy_(alone)
        torch.cuda.synchronize()
        model.step()
        gpu_ctx.synchronize()
        assert torch.equal(model.logits[b], got[b])
    model.close()


def test_a_served_run(gpu_ctx):
    """Steps, draws and evictions in one captured loop body, replayed token by token, against the
    same calls made one at a time; the budget holds and every sequence keeps its newest slots."""
    cfg, B, ctx_len, keep, recent, steps = LLAMA_TINY, 3, 48, 40, 8, 12

    def make():
        return dec.Decoder(cfg, gpu_ctx, B, ctx_len, max_new=16, seed=8, page_size=16, track=True)

    rng = np.random.default_rng(1)
    us = torch.from_numpy(rng.random((steps, B), dtype=np.float32)).cuda()
    first = torch.tensor([1, 2, 3], dtype=torch.int32)
    runs = []
    stream = torch.cuda.Stream()
    for captured in (False, True):
        model = make()
        u, since = torch.zeros(B, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
        temp, top_p = torch.full((B,), 0.8, device="cuda"), torch.full((B,), 0.9, device="cuda")
        prob = torch.zeros(B, device="cuda")
        model.tokens.copy_(first)
        torch.cuda.synchronize()
        gpu_ctx.set_stream(stream)

        def body():
            model.step()
            model.sample(u, temperature=temp, top_p=top_p, prob=prob)
            model.evict(keep, recent_from=since)

        try:
            with torch.cuda.stream(stream):
                seen, g = [], None
                if captured:
                    snapshot = [(L["k"].clone(), L["v"].clone(), L["mass"].clone(), L["slot_pos"].clone())
                                for L in model.layers]
                    since.copy_(model.positions - recent + 1)
                    body()  # sizes what is allocated at the first call
                    for L, old in zip(model.layers, snapshot):
                        for key, t in zip(("k", "v", "mass", "slot_pos"), old):
                            L[key].copy_(t)
                    model.tokens.copy_(first)
                    model.lens.fill_(ctx_len + 1)
                    stream.synchronize()
                    g = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(g, stream=stream):
                        body()
                for i in range(steps):
                    u.copy_(us[i])
                    since.copy_(model.positions - recent + 1)
                    g.replay() if captured else body()
                    stream.synchronize()
                    assert model.lens.tolist() == [keep] * B
                    for L in model.layers:
                        p = L["slot_pos"][:, :, :keep]
                        newest = int(model.positions[0])
                        for d in range(recent):
                            assert ((p == newest - d).sum(-1) == 1).all()
                    seen.append((model.tokens.tolist(), prob.tolist()))
                    model.lens.add_(1)
                    model.positions.add_(1)
                del g
            gpu_ctx.synchronize()
        finally:
            gpu_ctx.set_stream(None)
        runs.append(seen)
        assert all(0 <= t < cfg.vocab for toks, _ in seen for t in toks)
        model.close()
    assert runs[0] == runs[1]


def test_options_that_do_not_go_together(gpu_ctx):
    with pytest.raises(ValueError):
        dec.Decoder(LLAMA_TINY, gpu_ctx, 1, 8, page_size=16, step_kernel=True)
    with pytest.raises(ValueError):
        dec.Decoder(LLAMA_TINY, gpu_ctx, 1, 8, track=True)
    model = dec.Decoder(LLAMA_TINY, gpu_ctx, 1, 8, page_size=16)
    with pytest.raises(ValueError):
        model.evict(4)
    model.close()
