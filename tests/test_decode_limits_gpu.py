"""The decode-step operators at the edges of what their header allows."""
from __future__ import annotations

import math
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import decode as D
from softhier_cuda import decode, lib as L
from test_decode_gpu import DEV, Pool, _attn_tol, _i32, _np, _p

pytestmark = pytest.mark.gpu


# ---- softmax exponents far from zero -------------------------------------------------------------------------------------
def _offset_case(rt, fmt, dh, nq, big, max_q, seed=1):
    """The scores of a row share a large offset: column 0 of every key is 96, of every row +-`big`; the other columns are small
    whole numbers. All sums are whole numbers below 2^24 and the scales powers of two, so the scores themselves are exact.
    -> outputs, oracle's outputs, tolerance."""
    rng = np.random.default_rng(seed)
    H, heads, page = 4, 2, 32
    lens = np.array([300, 47 + nq])
    blocks = -(-lens // page)
    pages = int(blocks.sum())
    pool = Pool(pages, heads, page, dh, fmt, seed)
    k = rng.integers(-3, 4, pool.shape).astype(np.float64)
    k[..., 0] = 96
    pool.codes[0] = D.encode(k, fmt)
    pool.scales[0] = np.full((pages, heads), 2.0 ** -5, np.float32)
    pool.scales[1] = np.full((pages, heads), 2.0 ** -6, np.float32)
    raw = np.stack(pool.codes)
    pool.raw.copy_(torch.from_numpy(raw.reshape(-1)))
    for i in range(2):
        pool.dev_scales[i].copy_(torch.from_numpy(pool.scales[i]))
    table = np.zeros((2, int(blocks.max())), np.int64)
    table[0, :blocks[0]], table[1, :blocks[1]] = np.arange(blocks[0]), blocks[0] + np.arange(blocks[1])
    q_start = np.array([0, nq, 2 * nq])
    T = 2 * nq
    q = rng.integers(-2, 3, (T, H, dh)).astype(np.float16)
    q[:, :, 0] = big * np.where((np.arange(T)[:, None] + np.arange(H)) % 2, -1, 1)
    q = q.reshape(T, H * dh)
    scale = 2.0 ** (2 if dh == 64 else 1)
    dq, do, ws = torch.from_numpy(q).to(DEV), torch.zeros((T, H * dh), dtype=torch.float16, device=DEV), \
        torch.zeros(L.KV8_WS_BYTES, dtype=torch.uint8, device=DEV)
    d_table, d_lens, d_start = _i32(table), _i32(lens), _i32(q_start)
    assert rt.lib.sh_cuda_attention_kv8(_p(dq), _p(do), pool.handle, _p(d_table), table.shape[1], _p(d_lens), _p(d_start), 2, T,
                                        max_q, H, H * dh, H * dh, scale, _p(ws), ws.numel()) == 0
    rt.check()
    want, mean_abs, _, _ = D.attention_kv8(q, *pool.codes, *pool.scales, table, lens, q_start, H, scale, fmt)
    # Exponents of two of up to E = scale log2(e) (96 big + 2 * 3 * dh) 2^-5, each rounded twice on its way (its multiply-add; the
    # maximum that is taken off), in numerator and denominator: 4 half steps of 2^-24 E, times ln 2 < 1; 2^-21 for exp2 and
    # the products by the factors of a moved maximum; a half step of fp16 for the weights (2^-25 of the largest for those
    # below the normal range) and one for the output; fp32 sums over the keys.
    n = float(lens.max())
    E = scale * 1.4427 * (96 * big + 6 * dh) / 32 + 6
    vmax = np.abs(D.decode(pool.codes[1], fmt) * pool.scales[1][:, :, None, None]).max()
    tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + (2.0 ** -11 + 4 * 2.0 ** -24 * E + 2.0 ** -21 + 2 * n * 2.0 ** -24) * 1.01 * mean_abs \
        + n * 2.0 ** -25 * vmax
    return _np(do).astype(np.float64), want, tol


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("nq,max_q", [(1, 1), (30, 30), (80, 80), (1, 80)])
@pytest.mark.parametrize("big", [16, 180, 300, 2047])
def test_attention_depends_on_score_differences_only(gpu_lib, fmt, dh, nq, max_q, big):
    """Exponents of up to about +-280, 3100, 5200 and 35000 (half of that at dh = 128): the row's maximum is taken off whole,
    however large it is."""
    got, want, tol = _offset_case(gpu_lib, fmt, dh, nq, big, max_q)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])
    assert (np.abs(got).max(1) > 0).all()


# ---- tables: shared memory around 48 KiB ---------------------------------------------------------------------------------
@pytest.mark.parametrize("many_rows", [False, True])
def test_tables_of_sizes_around_48_kib_of_shared_memory(many_rows):
    """In a process of its own, as the border depends on what was called before."""
    worker = Path(__file__).resolve().parent / "tables_worker.py"
    r = subprocess.run([sys.executable, str(worker), "many" if many_rows else "few"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "OK" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]


# ---- lengths past the table -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("nq", [1, 3, 12, 80])
@pytest.mark.parametrize("over", [1, 2, 40, 1000, 2 ** 31 - 1 - 64])
def test_attention_of_a_length_past_the_table(gpu_lib, nq, over):
    """Row i attends the tokens j <= lens - n + i that the table has: of a length `over` past it the last `over` rows attend all of
    them, and the rows before as in a request of n - over rows that ends with the table."""
    rt = gpu_lib
    page, heads, dh, H, cap = 16, 2, 64, 4, 64
    pool = Pool(8, heads, page, dh, "int8", 4)
    table = np.array([[0, 1, 2, 3], [4, 5, 6, 7]])
    rng = np.random.default_rng(nq)
    q = rng.standard_normal((2 * nq, H * dh)).astype(np.float16)
    dq, do = torch.from_numpy(q).to(DEV), torch.zeros((2 * nq, H * dh), dtype=torch.float16, device=DEV)
    d = _i32(table), _i32([cap + over, 50]), _i32([0, nq, 2 * nq])
    ws = torch.zeros(L.KV8_WS_BYTES, dtype=torch.uint8, device=DEV)
    assert rt.lib.sh_cuda_attention_kv8(_p(dq), _p(do), pool.handle, _p(d[0]), 4, _p(d[1]), _p(d[2]), 2, 2 * nq, nq, H, H * dh, H * dh,
                                        0.125, _p(ws), ws.numel()) == 0
    assert rt.lib.sh_cuda_device_error() == 2
    early = max(nq - over, 0)
    starts, lens = [0], []
    if early:
        starts, lens = [0, early], [cap]
    for _ in range(early, nq):
        starts.append(starts[-1] + 1)
        lens.append(cap)
    starts.append(2 * nq)
    lens.append(50)
    rows = np.concatenate([np.repeat(table[:1], len(lens) - 1, 0), table[1:]])
    want, mean_abs, big, keys = D.attention_kv8(q, *pool.codes, *pool.scales, rows, lens, starts, H, 0.125, "int8")
    vmax = np.abs(D.decode(pool.codes[1], "int8") * pool.scales[1][:, :, None, None]).max()
    err = np.abs(_np(do).astype(np.float64) - want)
    tol = _attn_tol(want, mean_abs, big, keys, H, dh, vmax)
    assert (err <= tol).all(), np.argwhere(err > tol)[:4]


# ---- K and V far apart ----------------------------------------------------------------------------------------------------
class FarMemory:
    """`size` bytes of device memory at an address at least 2^41 bytes away from `other` (virtual memory management of the
    driver: reserve, create, map), as a second allocator may give them."""

    def __init__(self, size, other):
        import ctypes as C
        self.C, self.cu = C, C.CDLL("libcuda.so.1")

        class Location(C.Structure):
            _fields_ = [("type", C.c_int), ("id", C.c_int)]

        class Prop(C.Structure):
            _fields_ = [("type", C.c_int), ("handles", C.c_int), ("location", Location), ("win32", C.c_void_p),
                        ("flags", C.c_ubyte * 8)]

        class Access(C.Structure):
            _fields_ = [("location", Location), ("flags", C.c_int)]
        loc = Location(1, torch.cuda.current_device())             # a device, pinned memory, read and write
        self.ptr = self.handle = None
        self.size, self.reserved = -(-size // (1 << 21)) * (1 << 21), 1 << 30
        for hint in (0, 1 << 45, other - (1 << 42) >> 21 << 21):
            p = C.c_uint64()
            if self.cu.cuMemAddressReserve(C.byref(p), C.c_size_t(self.reserved), C.c_size_t(0), C.c_uint64(hint), C.c_ulonglong(0)):
                continue
            if abs(p.value - other) >= 1 << 41:
                self.ptr = p.value
                break
            self.cu.cuMemAddressFree(p, C.c_size_t(self.reserved))
        if self.ptr is None:
            pytest.skip("the driver gives no address that far away")
        h = C.c_uint64()
        assert self.cu.cuMemCreate(C.byref(h), C.c_size_t(self.size), C.byref(Prop(1, 0, loc)), C.c_ulonglong(0)) == 0
        self.handle = h
        assert self.cu.cuMemMap(C.c_uint64(self.ptr), C.c_size_t(self.size), C.c_size_t(0), h, C.c_ulonglong(0)) == 0
        assert self.cu.cuMemSetAccess(C.c_uint64(self.ptr), C.c_size_t(self.size), C.byref(Access(loc, 3)), C.c_size_t(1)) == 0

    def free(self):
        C = self.C
        torch.cuda.synchronize()
        assert self.cu.cuMemUnmap(C.c_uint64(self.ptr), C.c_size_t(self.size)) == 0
        assert self.cu.cuMemRelease(self.handle) == 0
        assert self.cu.cuMemAddressFree(C.c_uint64(self.ptr), C.c_size_t(self.reserved)) == 0


@pytest.mark.parametrize("fmt,page,dh", [("int8", 16, 64), ("fp8", 64, 64), ("fp8", 16, 128), ("int8", 128, 128)])
def test_attention_of_arrays_in_different_address_ranges(gpu_lib, fmt, page, dh):
    """K and V more than 2^40 bytes apart, either first: the bits of the same cache with both side by side."""
    rt = gpu_lib
    H, heads = 8, 2
    lens = np.array([300, 1, 77, 33])
    blocks = -(-lens // page)
    pool = Pool(int(blocks.sum()), heads, page, dh, fmt, 3)
    size = int(np.prod(pool.shape))
    table = np.zeros((4, int(blocks.max())), np.int64)
    for r in range(4):
        table[r, :blocks[r]] = blocks[:r].sum() + np.arange(blocks[r])
    far = FarMemory(size, _p(pool.raw))
    try:
        for near_k in (True, False):
            for nq in ((1, 1, 1, 1), (5, 1, 0, 7), (100, 1, 20, 33)):
                T, start = sum(nq), _i32(np.concatenate([[0], np.cumsum(nq)]))
                q = torch.randn((T, H * dh), device=DEV, generator=torch.Generator(DEV).manual_seed(T)).half()
                ws = torch.zeros(L.KV8_WS_BYTES, dtype=torch.uint8, device=DEV)
                d_table, d_lens, outs = _i32(table), _i32(lens), []
                for apart in (False, True):
                    k, v = _p(pool.raw), _p(pool.raw) + size
                    if apart:
                        src = v if near_k else k
                        assert rt.lib.sh_cuda_copy2d(far.ptr, size, src, size, size, 1, rt.lib.sh_cuda_get_stream()) == 0
                        k, v = (k, far.ptr) if near_k else (far.ptr, v)
                    h = L.Kv8(k, v, _p(pool.dev_scales[0]), _p(pool.dev_scales[1]), pool.stride, pool.shape[0], page, heads, dh,
                              decode.FORMATS[fmt])
                    o = torch.full_like(q, 7.0)
                    rc = rt.lib.sh_cuda_attention_kv8(_p(q), _p(o), h, _p(d_table), table.shape[1], _p(d_lens), _p(start), 4, T, max(nq),
                                                      H, H * dh, H * dh, 0.125, _p(ws), ws.numel())
                    assert rc == 0
                    rt.check()
                    outs.append(_np(o).view(np.uint16))
                np.testing.assert_array_equal(outs[0], outs[1])
    finally:
        far.free()


# ---- after a failed call ----------------------------------------------------------------------------------------------------
def test_append_after_a_failed_call(gpu_lib, capfd):
    """A CUDA call of the library that was refused before, and reported, is not reported as this one's."""
    rt = gpu_lib
    pool = Pool(4, 2, 16, 64, "int8", 2)
    x, s = torch.ones((1, 128), dtype=torch.float16, device=DEV), _i32([5])
    rt.check()
    assert not rt.lib.sh_cuda_ipc_alloc(1 << 50)           # more memory than there is
    assert rt.lib.sh_cuda_kv8_append(pool.handle, _p(x), _p(x), 1, 128, 128, _p(s)) == 0
    assert rt.lib.sh_cuda_last_error() != 0 and rt.lib.sh_cuda_last_error() == 0
    rt.check()
    capfd.readouterr()


# ---- queries that are not finite ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("nq", [1, 12, 80])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_attention_of_infinite_queries_is_nan_whatever_the_keys(gpu_lib, fmt, nq, value):
    """Also where every key has the same sign in that column, so that all scores are +infinity or all -infinity; a row without keys
    stays zero."""
    rt = gpu_lib
    pool = Pool(8, 2, 32, 64, fmt, 4)
    pool.codes[0][..., 9] = D.encode(np.array(3.0), fmt)
    pool.raw.copy_(torch.from_numpy(np.stack(pool.codes).reshape(-1)))
    q = torch.randn((2 * nq, 256), device=DEV, generator=torch.Generator(DEV).manual_seed(1)).half()
    start, table, lens = _i32([0, nq, 2 * nq]), _i32([[0, 1, 2, 3], [4, 5, 6, 7]]), _i32([nq - 1, 100])
    ws = torch.zeros(L.KV8_WS_BYTES, dtype=torch.uint8, device=DEV)

    def run(x):
        o = torch.zeros_like(x)
        assert rt.lib.sh_cuda_attention_kv8(_p(x), _p(o), pool.handle, _p(table), 4, _p(lens), _p(start), 2, 2 * nq, nq, 4, 256, 256,
                                            0.125, _p(ws), ws.numel()) == 0
        rt.check()
        return _np(o).reshape(2 * nq, 4, 64)
    good = run(q)
    rows = sorted({0, nq - 1, nq, 2 * nq - 1})
    x = q.clone()
    for r in rows:
        x[r, 64 + 9] = value
    got = run(x)
    hit = np.zeros(good.shape[:2], bool)
    for r in rows:
        hit[r, 1] = r > 0           # row 0 has no key
    assert np.isnan(got[hit]).all() and (got[0] == 0).all()
    assert np.array_equal(got[~hit].view(np.uint16), good[~hit].view(np.uint16))


# ---- the host side ------------------------------------------------------------------------------------------------------------
def test_cache_made_while_torchs_stream_is_busy(gpu_lib):
    """A new cache is used on another stream at once, while torch's own stream, which fills it, had work to do."""
    rt, old, side = gpu_lib, gpu_lib.stream, torch.cuda.Stream()
    add = _i32([3, 0, 2])
    torch.cuda.synchronize()
    try:
        rt.activate(side)
        torch.cuda._sleep(100_000_000)
        cache = decode.KvCache(rt, layers=1, heads=2, dh=64, page=16, pages=8, requests=3, blocks=2, t_cap=8)
        cache.step(add)
        rt.check()
    finally:
        rt.activate(old)
    torch.cuda.synchronize()
    assert cache.lens.tolist() == [3, 0, 2] and cache.pool[:3].tolist() == [2, 6, 0]
    assert cache.slots.tolist() == [0, 1, 2, 16, 17, -1, -1, -1]


# ---- the accuracy of the kernel for few rows ----------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("nq,max_q", [(1, 1), (12, 12), (40, 30)])
def test_attention_of_few_rows_is_off_by_its_outputs_rounding_only(gpu_lib, fmt, dh, nq, max_q):
    """Exact scores as above, without the offset. The weights go in as fp16 and the rest of that rounding (2^-22 of each, 2^-25 of
    the largest where the rest is below the normal range), so next to the output's half step only fp32 terms are left. Weights
    that are only rounded to fp16, planted in the oracle, are outside of the bound."""
    rng = np.random.default_rng(dh + nq)
    H, heads, page, n = 4, 2, 16, 60
    pool = Pool(4, heads, page, dh, fmt, 7)
    pool.codes[0] = D.encode(rng.integers(-3, 4, pool.shape).astype(np.float64), fmt)
    pool.scales = [np.full((4, heads), 2.0 ** -5, np.float32), np.full((4, heads), 2.0 ** -6, np.float32)]
    pool.raw.copy_(torch.from_numpy(np.stack(pool.codes).reshape(-1)))
    for i in range(2):
        pool.dev_scales[i].copy_(torch.from_numpy(pool.scales[i]))
    q = rng.integers(-2, 3, (nq, H * dh)).astype(np.float16)
    scale, table = 2.0, np.arange(4)[None]
    dq, do = torch.from_numpy(q).to(DEV), torch.zeros((nq, H * dh), dtype=torch.float16, device=DEV)
    ws, d = torch.zeros(L.KV8_WS_BYTES, dtype=torch.uint8, device=DEV), (_i32(table), _i32([n]), _i32([0, nq]))
    assert gpu_lib.lib.sh_cuda_attention_kv8(_p(dq), _p(do), pool.handle, _p(d[0]), 4, _p(d[1]), _p(d[2]), 1, nq, max_q, H, H * dh,
                                             H * dh, scale, _p(ws), ws.numel()) == 0
    gpu_lib.check()
    want, mean_abs, _, _ = D.attention_kv8(q, *pool.codes, *pool.scales, table, [n], [0, nq], H, scale, fmt)
    # as in _offset_case, with the weights' rounding as said above
    E = scale * 1.4427 * 6 * dh / 32 + 6
    v = D.decode(pool.codes[1], fmt) * 2.0 ** -6
    tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + n * 2.0 ** -25 * np.abs(v).max() \
        + (2.0 ** -22 + 4 * 2.0 ** -24 * E + 2.0 ** -21 + 2 * n * 2.0 ** -24) * 1.01 * mean_abs
    err = np.abs(_np(do).astype(np.float64) - want)
    assert (err <= tol).all(), float((err / tol).max())
    planted = np.zeros_like(want)
    k = D.decode(pool.codes[0], fmt) * 2.0 ** -5
    for i in range(nq):
        for h in range(H):
            keys = k[:, h // 2].reshape(-1, dh)[:n - nq + i + 1]
            x = scale * (keys @ q[i, h * dh:(h + 1) * dh].astype(np.float64))
            w = np.exp(x - x.max())
            planted[i, h * dh:(h + 1) * dh] = w.astype(np.float16).astype(np.float64) @ v[:, h // 2].reshape(-1, dh)[:len(keys)] / w.sum()
    assert (np.abs(planted.astype(np.float16).astype(np.float64) - want) > tol).any()
