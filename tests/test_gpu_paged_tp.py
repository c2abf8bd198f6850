"""A tensor-parallel decoder on a paged cache, one process per GPU, against the same
decoder on one GPU: sequences at positions of their own, an eviction between
steps.  Skipped with fewer than 2 GPUs; tests/test_paged_tp_host.py covers what
each form queues without one."""
import os

import pytest

from test_gpu_decoder import LLAMA_TINY, LLAMA_TINY_TP, TOL, _free_port, _gpus, rel_err

pytestmark = pytest.mark.gpu


def _worker(rank, world, port, out_dir):
    import datetime
    import numpy as np
    import torch
    import torch.distributed as dist
    from pesti_b200 import decoder as dec
    from pesti_b200 import kq
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    torch.cuda.set_device(rank)
    dist.init_process_group("gloo", rank=rank, world_size=world, timeout=datetime.timedelta(seconds=60))
    status = "ok"
    try:
        ctx = kq.Context(rank)
        for cfg in (LLAMA_TINY, LLAMA_TINY_TP):
            tp = kq.TensorParallel(ctx, world, rank, max_out_elems=dec.exchange_elems(cfg, 2))
            for batch in (1, 2):
                sizes = dict(max_new=3, seed=7, page_size=16, track=True)
                model = dec.Decoder(cfg, ctx, batch, 20, world=world, rank=rank, tp=tp, **sizes)
                single = dec.Decoder(cfg, ctx, batch, 20, **sizes)
                for pos in (20, 21):  # two steps: the exchange slots alternate
                    lens = [pos + 1, pos - 9][:batch]
                    for m in (model, single):
                        m.tokens.copy_(torch.tensor([4 + pos, 5][:batch], dtype=torch.int32))
                        m.lens.copy_(torch.tensor(lens, dtype=torch.int32))
                        m.positions.copy_(m.lens - 1)
                        torch.cuda.synchronize()
                        m.step()
                    ctx.synchronize()
                    a, b = model.logits.cpu().numpy(), single.logits.cpu().numpy()
                    # the exchanged parts and the split of the attention round otherwise than one
                    # GPU's: half of the decoder tests' bound against the oracle
                    if status == "ok" and not (np.isfinite(a).all() and rel_err(a, b) <= TOL / 2):
                        status = f"{cfg.name} batch {batch} pos {pos}: logits differ by {rel_err(a, b):.2e}"
                model.evict(12)
                ctx.synchronize()
                if status == "ok" and model.lens.tolist() != [12, 12][:batch]:
                    status = f"{cfg.name} batch {batch}: {model.lens.tolist()} slots after the eviction"
                model.close()
                single.close()
            tp.close()
        ctx.close()
    except Exception as e:  # report to the parent
        status = f"exception: {e!r}"
    finally:
        with open(os.path.join(out_dir, f"r{rank}"), "w") as fh:
            fh.write(status)
        dist.destroy_process_group()


@pytest.mark.skipif(_gpus() < 2, reason="needs 2 GPUs")
def test_paged_decode_on_two_gpus_matches_one(tmp_path):
    import torch.multiprocessing as mp
    mp.start_processes(_worker, args=(2, _free_port(), str(tmp_path)), nprocs=2, start_method="spawn", join=True)
    for r in range(2):
        assert (tmp_path / f"r{r}").read_text() == "ok", f"rank {r}"
