"""The decode-step operators without a GPU: refusals (checked before any CUDA call), the 4-bit quantiser, the oracle."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import decode as D
from softhier_cuda import decode, lib as L

A = 1 << 20          # an address that is only looked at, never followed


@pytest.fixture(scope="module")
def lib():
    if not L.LIB_PATH.exists():
        import __graft_entry__
        __graft_entry__.build()
    return L.load()


def _cache(**kw):
    f = dict(k=A, v=A, k_scale=A, v_scale=A, page_stride=4 * 16 * 64, pages=8, page=16, heads=4, dh=64, fmt=L.SH_INT8)
    f.update(kw)
    return L.Kv8(*[f[n] for n, _ in L.Kv8._fields_])


def _attn(lib, cache, **kw):
    f = dict(q=A, o=A, table=A, ld_table=8, lens=A, q_start=A, R=2, T=2, max_q=1, H=8, ldq=512, ldo=512, scale=0.125, ws=A,
             ws_bytes=L.KV8_WS_BYTES)
    f.update(kw)
    return lib.sh_cuda_attention_kv8(f["q"], f["o"], cache, *[f[n] for n in (
        "table", "ld_table", "lens", "q_start", "R", "T", "max_q", "H", "ldq", "ldo", "scale", "ws", "ws_bytes")])


BAD_CACHE = [dict(k=0), dict(v=0), dict(k_scale=0), dict(v_scale=2), dict(k=A + 8), dict(page=24), dict(page=256), dict(dh=80),
             dict(heads=0), dict(pages=0), dict(pages=1 << 27), dict(page_stride=4 * 16 * 64 - 16),
             dict(page_stride=4 * 16 * 64 + 8)]


@pytest.mark.parametrize("kw", BAD_CACHE, ids=str)
def test_bad_caches_are_refused(lib, capfd, kw):
    lib.sh_cuda_last_error()
    assert lib.sh_cuda_kv8_append(_cache(**kw), A, A, 1, 256, 256, A) == -1
    assert _attn(lib, _cache(**kw)) == -1
    out = capfd.readouterr().out
    assert "[sh_cuda_kv8_append]" in out and "[sh_cuda_attention_kv8]" in out
    assert lib.sh_cuda_last_error() == -1


def test_other_formats_are_refused(lib, capfd):
    lib.sh_cuda_last_error()
    for fmt in (L.SH_FP16, L.SH_INT16, 9):
        assert lib.sh_cuda_kv8_append(_cache(fmt=fmt), A, A, 1, 256, 256, A) == -3
        assert _attn(lib, _cache(fmt=fmt)) == -3
    assert lib.sh_cuda_kv8_append(None, A, A, 1, 256, 256, A) == -1
    assert lib.sh_cuda_last_error() == -3
    capfd.readouterr()


def test_append_and_attention_refusals(lib, capfd):
    lib.sh_cuda_last_error()
    for args in ((0, A, 1, 256, 256, A), (A, 0, 1, 256, 256, A), (A, A, 1, 255, 256, A), (A, A, 1, 256, 255, A),
                 (A, A, 1, 256, 256, 0), (A + 1, A, 1, 256, 256, A), (A, A, 1 << 31, 256, 256, A),
                 (A, A, 1, 256, 256, A + 2)):
        assert lib.sh_cuda_kv8_append(_cache(), *args) == -1, args
    assert lib.sh_cuda_kv8_append(_cache(), 0, 0, 0, 256, 256, 0) == 0           # no rows: nothing to do
    for kw in (dict(H=6), dict(H=0), dict(ldq=511), dict(ldo=511), dict(q=0), dict(o=0), dict(q=A + 1), dict(table=0),
               dict(lens=0), dict(q_start=0), dict(ld_table=0), dict(ld_table=1 << 27), dict(scale=float("nan")),
               dict(scale=float("inf")), dict(ws=0), dict(ws=A + 4), dict(ws_bytes=L.KV8_WS_BYTES - 1), dict(T=1 << 29),
               dict(table=A + 2), dict(lens=A + 1), dict(q_start=A + 3)):
        assert _attn(lib, _cache(), **kw) == -1, kw
    assert _attn(lib, _cache(), R=0) == 0 and _attn(lib, _cache(), T=0) == 0
    lib.sh_cuda_last_error()
    capfd.readouterr()


def test_tables_refusals(lib, capfd):
    lib.sh_cuda_last_error()
    good = dict(lens=A, add=A, R=4, page=16, table=A, ld_table=8, ring=A, pages=64, pool=A, pool_out=A, lens_out=A, q_start=A,
                slots=A, pos=A, t_cap=64)
    for kw in (dict(page=8), dict(page=0), dict(page=48), dict(pages=0), dict(pages=1 << 27), dict(R=8193), dict(lens=0),
               dict(add=0), dict(table=0), dict(ring=0), dict(pool=0), dict(pool_out=0), dict(lens_out=0), dict(q_start=0),
               dict(slots=0), dict(pos=0), dict(ld_table=0), dict(ld_table=1 << 27), dict(t_cap=1 << 31),
               *({name: A + 2} for name in good if good[name] == A)):
        assert lib.sh_cuda_kv_tables(*(good | kw).values()) == -1, kw
    assert lib.sh_cuda_kv_tables(*(good | dict(R=0)).values()) == 0
    assert "[sh_cuda_kv_tables]" in capfd.readouterr().out
    lib.sh_cuda_last_error()


def test_gemv_w4_refusals(lib, capfd):
    lib.sh_cuda_last_error()
    good = dict(x=A, codes=A, scales=A, zeros=0, z=A, M=4, N=64, K=256, ldx=256, ldw=128, ldz=64, group=64, bias=0, residual=0,
                ldr=0, flags=0)
    for kw in (dict(M=33), dict(group=16), dict(group=256), dict(K=224), dict(K=0),
               dict(K=(1 << 18) + 64, ldx=1 << 20, ldw=1 << 19), dict(ldx=255), dict(ldz=63), dict(ldw=112),
               dict(ldw=136), dict(x=0), dict(codes=0), dict(codes=A + 8), dict(scales=0), dict(z=0), dict(x=A + 1),
               dict(flags=L.EPI_BIAS), dict(flags=L.EPI_RESIDUAL), dict(flags=L.EPI_RESIDUAL, residual=A, ldr=63),
               dict(flags=L.EPI_GELU), dict(flags=L.EPI_ACCUMULATE)):
        assert lib.sh_cuda_gemv_w4(*(good | kw).values()) == -1, kw
    assert lib.sh_cuda_gemv_w4(*(good | dict(M=0)).values()) == 0 and lib.sh_cuda_gemv_w4(*(good | dict(N=0)).values()) == 0
    assert "[sh_cuda_gemv_w4]" in capfd.readouterr().out
    lib.sh_cuda_last_error()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("symmetric", [False, True])
def test_quantize_w4_is_within_a_step(group, symmetric):
    """Each value lies within the range that its group's steps cover, so it is off by at most half a step, plus the range's
    end when the fp16 scale was rounded down (15 steps of 2^-11), plus half a step of the rounded zero point."""
    rng = np.random.default_rng(3)
    w = rng.standard_normal((256, 40)).astype(np.float32)
    w[:group, 3] = 0.0                                     # a group without a value
    codes, scales, zeros = decode.quantize_w4(w, group, symmetric)
    assert codes.shape == (40, 128) and (zeros is None) == symmetric
    assert all(a is None or a.flags.c_contiguous for a in (codes, scales, zeros))      # their addresses go to the library
    back = D.w4_weights(codes, scales, zeros, group, 256)
    step = np.repeat(scales.astype(np.float64), group, 1).T
    assert np.all(np.abs(back - w) <= step * (1.0 + 15 * 2.0 ** -11) + 1e-12)
    assert np.all(back[:group, 3] == 0)
    with pytest.raises(ValueError):
        decode.quantize_w4(w, 96)
    for x in (np.nan, np.inf, 1e7):                        # no fp16 scale
        w[5, 5] = x
        with pytest.raises(ValueError):
            decode.quantize_w4(w, group, symmetric)


def test_oracle_e4m3_agrees_with_torch():
    import torch
    codes = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(codes).view(torch.float8_e4m3fn).float().numpy()
    np.testing.assert_array_equal(D.e4m3_values(), want.astype(np.float64))
    y = np.concatenate([np.random.default_rng(1).standard_normal(20000) * 40, np.linspace(-448, 448, 7169),
                        np.random.default_rng(2).standard_normal(5000) * 0.01]).astype(np.float32)
    got = D.decode(D.e4m3_encode(y), "fp8")
    np.testing.assert_array_equal(got, torch.from_numpy(y).to(torch.float8_e4m3fn).double().numpy())


def test_quotients_by_eight_bit_scales_never_sit_near_a_border():
    """Codes from 32-bit and 64-bit division are the same, for every fp16 magnitude against random 8-bit scales."""
    x = np.arange(1, 0x7C00, dtype=np.uint16).view(np.float16)
    rng = np.random.default_rng(4)
    for fmt in ("int8", "fp8"):
        for top in rng.choice(x, 40):
            s = D.up8(float(top) / D.QMAX[fmt])
            v = x[x <= top]
            a = (v.astype(np.float32) / np.float32(s)).astype(np.float64)
            np.testing.assert_array_equal(D.encode(a, fmt), D.encode(v.astype(np.float64) / s, fmt))
            assert float(np.float32(s)) == s
