"""The next tokens from a decoder's logits (kq_dec_sample, include/pesti_decoder.h)."""
from __future__ import annotations

import ctypes

from . import kq


def _bind(lib: ctypes.CDLL) -> ctypes.CDLL:
    if lib.kq_dec_sample.argtypes is None:
        P, I64 = ctypes.c_void_p, ctypes.c_int64
        lib.kq_dec_sample.restype = ctypes.c_int
        lib.kq_dec_sample.argtypes = [P, P, I64, I64, I64, P, P, P, P, P, P, P, P]
    return lib


def sample(ctx: "kq.Context", logits, u, tokens, *, temperature=None, top_k=None, top_p=None, min_p=None, prob=None,
           kept=None) -> None:
    """tokens[b] from logits [batch][vocab] (f32 rows) and uniform random
    numbers u[b] in [0, 1): temperature (<= 0: the greatest logit), then top_k
    (<= 0: all), top_p and min_p, each a [batch] vector or None.  prob receives
    the token's probability among the tokens kept, kept their number.  A row
    without a finite or +inf logit gives -1.  CUDA tensors on the context's
    device; queued on its stream."""
    import torch
    f32, i32, index = torch.float32, torch.int32, ctx.device
    shape, stride = logits.shape, logits.stride()
    if logits.dtype is not f32 or logits.get_device() != index or len(shape) != 2 or (stride[1] != 1 and shape[1] > 1):
        raise kq.KqError(kq.KQ_ERR_INVALID_ARG, f"logits: {logits.dtype} {tuple(shape)} strides {stride} on "
                         f"{logits.device}; rows of float32 on cuda:{index} are wanted")
    batch, vocab = shape
    want = (batch,)

    def ptr(t, name, dtype):
        if t is None:
            return None
        if t.dtype is not dtype or t.get_device() != index or t.shape != want or not t.is_contiguous():
            raise kq.KqError(kq.KQ_ERR_INVALID_ARG, f"{name}: {t.dtype} {tuple(t.shape)} on {t.device}; {batch} "
                             f"contiguous {dtype} on cuda:{index} are wanted")
        return t.data_ptr()

    rc = _bind(ctx.lib).kq_dec_sample(
        ctx.handle, logits.data_ptr(), stride[0] if batch > 1 else vocab, batch, vocab,
        ptr(temperature, "temperature", f32), ptr(top_k, "top_k", i32), ptr(top_p, "top_p", f32),
        ptr(min_p, "min_p", f32), ptr(u, "u", f32), ptr(tokens, "tokens", i32), ptr(prob, "prob", f32),
        ptr(kept, "kept", i32))
    if rc:
        ctx.check(rc, "kq_dec_sample")
