"""The paged cache and sampling without a GPU: null handles and tensors that do
not fit are refused before any device work, and the address arithmetic of the
kernels (kq_paged.cuh compiled for the host) holds at its borders."""
import ctypes
import os
import subprocess
import types

import pytest
import torch

from pesti_b200 import build, kq, paged, sampling

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    build.build()
    lib = kq.load_library()
    paged._bind(lib)
    sampling._bind(lib)
    return lib


def test_null_handles_are_refused(lib):
    P = ctypes.c_void_p
    out = P()
    assert lib.kq_kv_create(None, None, None, 1, 1, 16, 1, 64, ctypes.byref(out)) == kq.KQ_ERR_INVALID_ARG
    assert lib.kq_kv_destroy(None) == kq.KQ_ERR_INVALID_ARG
    assert lib.kq_kv_append(None, None, 0, 0, 1, None, None, None, None, 0, 0, 1.0, None, 0, None,
                            0) == kq.KQ_ERR_INVALID_ARG
    assert lib.kq_kv_attention_scratch(None, 1, 1, 0) == 0
    assert lib.kq_kv_attention(None, None, 0, None, 0, 1, 1, None, 1, None, None, 0, None, 0) == kq.KQ_ERR_INVALID_ARG
    assert lib.kq_kv_rope_attention(None, None, 0, None, 0, 1, 1, None, 1, None, None, 1.0, None, None, 0, None,
                                    0) == kq.KQ_ERR_INVALID_ARG
    assert lib.kq_kv_evict_scratch(None, 1, 1) == 0
    assert lib.kq_kv_evict(None, 1, None, 1, None, None, None, None, None, None, 1, None, 1, None,
                           0) == kq.KQ_ERR_INVALID_ARG
    assert lib.kq_dec_sample(None, None, 1, 1, 1, None, None, None, None, None, None, None,
                             None) == kq.KQ_ERR_INVALID_ARG


@pytest.mark.parametrize("k,v", [
    (torch.zeros(2, 1, 16, 64), torch.zeros(2, 1, 16, 64)),                              # not f16
    (torch.zeros(2, 1, 16, 64).half(), torch.zeros(3, 1, 16, 64).half()),                # two shapes
    (torch.zeros(2, 16, 64).half(), torch.zeros(2, 16, 64).half()),                      # three dimensions
    (torch.zeros(2, 16, 1, 64).half().transpose(1, 2), torch.zeros(2, 16, 1, 64).half().transpose(1, 2)[:, :, :8]),
    (torch.zeros(2, 1, 16, 64).half(), torch.zeros(2, 1, 16, 64).half()),                # not on the GPU
    (torch.zeros(2, 4, 16, 64).half().transpose(1, 2), torch.zeros(2, 4, 16, 64).half().transpose(1, 2)),  # strides
])
def test_pools_that_do_not_fit_are_refused(k, v):
    ctx = types.SimpleNamespace(device=0, lib=None)
    with pytest.raises(kq.KqError) as e:
        paged.PagedCache(ctx, k, v)
    assert e.value.status == kq.KQ_ERR_INVALID_ARG


def test_logits_off_the_gpu_are_refused():
    ctx = types.SimpleNamespace(device=0, lib=None)
    t = torch.zeros(1)
    with pytest.raises(kq.KqError) as e:
        sampling.sample(ctx, torch.zeros(1, 8), t, t.int())
    assert e.value.status == kq.KQ_ERR_INVALID_ARG


HOST = r"""
#include "kq_paged.cuh"
#include <cstdio>
#define CHECK(x) if (!(x)) { std::printf("%s\n", #x); return 1; }
using namespace kq;
int main() {
  KvPool p;
  p.pages = 70000; p.page_ld = 8 * 64 * 128; p.page_size = 64; p.hkv = 8; p.hd = 128;
  CHECK(kv_row(p, 0, 0, 0) == 0);
  CHECK(kv_row(p, 1, 65, 2) == 65536 + (2 * 64 + 1) * 128);
  CHECK(kv_row(p, 69999, 63, 7) == 70000ll * 65536 - 128);   // the last row of the pool, past 2^32 elements
  CHECK(kv_row(p, 70000, 0, 0) == -1);
  CHECK(kv_row(p, -1, 0, 0) == -1);
  CHECK(kv_row(p, 0x7fffffff, 0, 0) == -1);
  CHECK(kv_row(p, (int)0x80000000, 0, 0) == -1);
  bool bad;
  CHECK(kv_len(0, 100, &bad) == 0 && !bad);
  CHECK(kv_len(100, 100, &bad) == 100 && !bad);
  CHECK(kv_len(101, 100, &bad) == 0 && bad);
  CHECK(kv_len(-1, 100, &bad) == 0 && bad);
  CHECK(kv_len(0x7fffffff, 1ll << 40, &bad) == 0x7fffffff && !bad);
  const int sizes[][2] = {{16, 16}, {32, 32}, {48, 16}, {64, 64}, {96, 32}, {128, 64}, {1024, 64}, {1008, 16}};
  for (auto& s : sizes) CHECK(kv_box_rows(s[0]) == s[1]);
  return 0;
}
"""


def test_address_arithmetic_on_the_host(tmp_path):
    src, exe = tmp_path / "host.cpp", tmp_path / "host"
    src.write_text(HOST)
    cuda = os.path.dirname(os.path.dirname(build._nvcc()))
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "pesti_b200", "csrc"), "-I",
                    os.path.join(cuda, "include"), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
