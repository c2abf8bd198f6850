"""The tensor-parallel step forms on a paged cache, without a GPU: what a step
queues, in order, recorded from stand-ins for the library, the cache and the
group.  Each layer attends once, over this rank's heads, into the buffer that the
form's exchange reads; on a contiguous cache the older call stands in its place."""
import types

import pytest
import torch

from pesti_b200 import decoder as dec

CFG = dec.DecoderConfig("two-rank-tiny", 2, 512, 4, 2, 128, 1024, 300, 1e-5, 5e5, False)


class Recorder:
    """Any method notes its name and arguments; status codes are 0."""

    def __init__(self, log, prefix=""):
        self._log, self._prefix, self.handle = log, prefix, 7

    def __getattr__(self, name):
        def call(*args, **kwargs):
            self._log.append((self._prefix + name, args, kwargs))
            return 0
        return call


def rank_model(form, page_size):
    """One rank of two, with everything that step() touches."""
    log = []
    m = object.__new__(dec.Decoder)
    m.cfg, m.world, m.rank, m.batch = CFG, 2, 1, 1 if form == "column" else 2
    m.hq, m.hkv, hd = CFG.heads // 2, CFG.kv_heads // 2, CFG.head_dim
    m.lib, m.tp = Recorder(log), Recorder(log, "tp.")
    m.ctx = types.SimpleNamespace(handle=1, check=lambda rc, what: None)
    m.step_kernel = m.prefetch = m.fuse_batch = False
    m.col_split, m.col_batch, m.fused = form == "column", form == "column batch", form == "column"
    m.fused_attention, m.swiglu_mode, m.max_seq = True, dec.SWIGLU_REFERENCE, 32
    m.Dp = m.Ap = 512
    m.o_rows, m.f_rows, m.v_rows = (256, 512), (512, 1024), (150, 300)
    m.qkv_ld = (m.hq + 2 * m.hkv) * hd
    for name, cols in (("h", 512), ("h2", 512), ("a", 512), ("qkv", m.qkv_ld), ("attn", 512), ("attn_r", m.hq * hd),
                       ("o", 256), ("gu", 1024), ("s_r", 512), ("s", 1024), ("dn", 256), ("part", 512),
                       ("logits_r", 150), ("logits", 300), ("embed", 512)):
        setattr(m, name, torch.zeros(m.batch, cols))
    m.tokens, m.final_norm = torch.zeros(m.batch, dtype=torch.int32), None
    m.att_scratch, m.att_scratch_bytes = torch.zeros(1), 4
    m.page_size, m.track = page_size, True
    m.table, m.lens, m.positions, m.kv_scratch = (torch.zeros(1) for _ in range(4))
    m.head = Recorder(log, "head.")
    m.layers = [dict({k: Recorder(log, f"{k}.") for k in ("qkv", "o", "gu", "down")}, cache=Recorder(log, "cache."),
                     attn_norm=torch.ones(512), ffn_norm=torch.ones(512), k=torch.zeros(1), v=torch.zeros(1),
                     mass=torch.zeros(1), slot_pos=torch.zeros(1)) for _ in range(CFG.layers)]
    return m, log


@pytest.mark.parametrize("form", ["row gathers", "column batch", "column"])
def test_every_form_attends_over_the_pages(form):
    m, log = rank_model(form, 16)
    m.step()
    names = [n for n, _, _ in log]
    assert names.count("cache.rope_attention") == CFG.layers
    assert not any("kq_dec_rope" in n or "kq_dec_attention" in n for n in names)
    calls = [(a, k) for n, a, k in log if n == "cache.rope_attention"]
    for L, (args, kwargs) in zip(m.layers, calls):
        assert [id(t) for t in args] == [id(t) for t in (m.qkv, m.table, m.lens, m.attn_r, m.kv_scratch)]
        assert kwargs["theta"] == CFG.theta and kwargs["pos"] is m.positions
        assert kwargs["mass"] is L["mass"] and kwargs["slot_pos"] is L["slot_pos"]
    # the exchange that follows the attention reads what it wrote
    after = names[names.index("cache.rope_attention") + 1]
    assert after == {"row gathers": "tp.allgather", "column batch": "o.linear", "column": "kq_dec_tp_partial_linear"}[form]
    with pytest.raises(ValueError):
        m.step(3)


@pytest.mark.parametrize("form", ["row gathers", "column batch", "column"])
def test_only_the_attention_differs_from_the_contiguous_cache(form):
    paged, plog = rank_model(form, 16)
    plain, clog = rank_model(form, 0)
    paged.step()
    plain.step(20)
    swap = {"cache.rope_attention": "kq_dec_rope_attention"}
    assert [swap.get(n, n) for n, _, _ in plog] == [n for n, _, _ in clog]
    pos = [a[11] for n, a, _ in clog if n == "kq_dec_rope_attention"]
    assert pos == [20] * CFG.layers
    with pytest.raises(ValueError):
        plain.step()
