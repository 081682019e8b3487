"""Limits of the decode-step operators that need no GPU: what is refused before any CUDA call, and what their sources must hold."""
from __future__ import annotations

from pathlib import Path
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from oracle import decode as D
from softhier_cuda import decode, lib as L
from test_decode_cpu import _attn, _cache, lib  # noqa: F401  (lib: the fixture)

CSRC = Path(__file__).resolve().parents[1] / "softhier-mlir_b200" / "csrc"


@pytest.mark.parametrize("page", [16, 128])
def test_attention_refuses_tables_whose_tokens_pass_31_bits(lib, capfd, page):      # noqa: F811
    """Token numbers run ahead of a request's last one, so a table has to end 2^14 tokens before 2^31."""
    lib.sh_cuda_last_error()
    most = ((1 << 31) - (1 << 14)) // page
    cache = _cache(page=page, page_stride=4 * page * 64)
    for ld_table, T in ((most, 1), (most + 1, 0), (most - 8, 1 << 27), ((1 << 31) // page - 1, 0), ((1 << 32) // page, 0)):
        assert _attn(lib, cache, ld_table=ld_table, T=T, H=4, ldq=256, ldo=256) == -1, (ld_table, T)
        assert "need H a multiple" in capfd.readouterr().out
    assert _attn(lib, cache, ld_table=most, T=0) == 0
    lib.sh_cuda_last_error()
    capfd.readouterr()


@pytest.mark.parametrize("name", ["sh_kvcache.cu", "sh_attention_kv8.cu", "sh_gemv_w4.cu"])
def test_decode_kernels_read_what_predecessors_write_with_plain_loads(name):
    """Each operator of a step reads what the one before it wrote, and may be launched while that one still runs: loads that
    promise constant data for the kernel's whole life have no place there."""
    src = (CSRC / name).read_text()
    assert "__ldg(" not in src and "ld.global.nc" not in src and "__restrict__" not in src


def test_the_copy_warp_stores_a_stages_flags_before_an_arrival_that_releases_them():
    """cp.async.mbarrier.arrive tracks copies, not the thread's own stores: the flags that the converting warps read go before
    the arrival of lane 0, with the warp's barrier between."""
    src = (CSRC / "sh_attention_kv8.cu").read_text()
    warp = src[src.index("// ---------------- copies"):src.index("// ---------------- MMA issue")]
    store, arrive = warp.index("info[2] = ok"), warp.index("mbar_arrive_expect_tx(")
    assert warp.index("mbar_wait(c_empty") < store < warp.index("__syncwarp()", store) < arrive < warp.index("cp_async_arrive(")


@pytest.mark.parametrize("name", ["sh_kvcache.cu", "sh_attention_kv8.cu", "sh_gemv_w4.cu", "sh_kv8.cuh"])
def test_what_decode_calls_remember_per_device_is_atomic(name):
    """Several host threads may make their first calls at the same time."""
    lines = [ln.strip() for ln in (CSRC / name).read_text().splitlines()]
    kept = [ln for ln in lines if ln.startswith("static ") and "static_assert" not in ln and "constexpr" not in ln]
    assert all("std::atomic<" in ln for ln in kept), kept


def test_cluster_counts_are_kept_per_kernel_and_only_when_the_runtime_gave_them():
    """All forms of the kernel have one function type, so a table in a function over that type would be one for all of them."""
    src = (CSRC / "sh_gemv_w4.cu").read_text()
    fn = src[src.index("w4_clusters(") - 40:src.index("cudaError_t w4_try")]
    assert "template <auto Kernel>" in fn and fn.count(".store(") == 1
    failed = fn.index("!= cudaSuccess")
    assert failed < fn.index("return sms / s;", failed) < fn.index(".store(")


def test_a_cache_is_filled_before_and_used_on_its_own_device(monkeypatch):
    """The tensors are filled on torch's stream and used on the library's: the constructor waits for them. A call that finds another
    device current (a second runtime's) is made on the cache's."""
    now, waits, calls = [1], [], []

    class Device:
        def __init__(self, d):
            self.d = d

        def __enter__(self):
            self.old, now[0] = now[0], self.d

        def __exit__(self, *exc):
            now[0] = self.old

    for name in ("zeros", "arange"):
        make = getattr(torch, name)
        monkeypatch.setattr(torch, name, lambda *a, make=make, device=None, **k: make(*a, **k))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda d=None: waits.append((d, len(calls))))
    lib_ = SimpleNamespace(**{n: (lambda *a, n=n: calls.append((n, now[0])) or 0) for n in (
        "sh_cuda_kv_tables", "sh_cuda_kv8_append", "sh_cuda_attention_kv8")})
    cache = decode.KvCache(SimpleNamespace(device=0, lib=lib_), layers=1, heads=2, dh=64, page=16, pages=8, requests=3, blocks=2)
    assert waits == [(0, 0)]
    for current in (1, 0):
        now[0] = current
        cache.step(torch.ones(3, dtype=torch.int32))
        cache.append(0, 256, 256, 128, 128, 3)
        cache.attend(0, 256, 256, 3, 4, 256, 256, 0.125)
        assert now[0] == current
    assert [d for _, d in calls] == [0] * 6 and len({n for n, _ in calls}) == 3


@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-5, 1e-6, 2e-7, 1e-7, 1e-8])
@pytest.mark.parametrize("symmetric", [False, True])
def test_quantize_w4_covers_groups_of_tiny_weights(size, symmetric):
    """Scales below fp16's normal range (2^-14): half a step for the value, half a step for the zero point, and the end of the range
    when a normal scale was rounded down (15 steps of 2^-11)."""
    w = (np.random.default_rng(3).standard_normal((256, 40)) * size).astype(np.float32)
    w[:64, 3] = 0.0
    codes, scales, zeros = decode.quantize_w4(w, 64, symmetric)
    back = D.w4_weights(codes, scales, zeros, 64, 256)
    step = np.repeat(scales.astype(np.float64), 64, 1).T
    assert np.all(np.abs(back - w) <= step * (1.0 + 15 * 2.0 ** -11))
    assert scales.dtype == np.float16 and scales.flags.c_contiguous
    assert scales[3, 0] == 0 and np.all(back[:64, 3] == 0) and (np.delete(scales.reshape(-1), 12) > 0).all()
