"""The decode-step operators on the GPU (block tables, 8-bit K / V cache append and attention, 4-bit products) against the
64-bit oracle (oracle/decode.py), and a run of them together."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import decode as D, llm
from softhier_cuda import decode, lib as L
from softhier_cuda.runtime import ShCudaError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
A = 0xFFFFFFFF


def _p(t):
    return t.data_ptr()


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)


def _np(t):
    return t.cpu().numpy()


# ---- tables ------------------------------------------------------------------------------------------------------------
def _tables_case(lens, add, page, ld, spare, seed, head=None):
    rng = np.random.default_rng(seed)
    lens, add = np.asarray(lens), np.asarray(add)
    have = -(-lens // page)
    used = int(have.sum())
    pages = used + spare
    ids = rng.permutation(pages)
    table = np.full((lens.size, ld), -7, np.int64)
    at = 0
    for r in range(lens.size):
        table[r, :have[r]] = ids[at:at + have[r]]
        at += have[r]
    ring = np.full(pages, -9, np.int64)
    head = int(rng.integers(pages)) if head is None else head
    ring[(head + np.arange(spare)) % pages] = ids[used:]
    return lens, add, table, ring, np.array([head, spare, 0, 0, 0, 0, 0, 0])


def _run_tables(rt, lens, add, page, table, ring, pool, t_cap, in_place, offset=0):
    d = {"lens": _i32(lens), "add": _i32(add), "table": _i32(table), "ring": _i32(ring), "pool": _i32(pool)}
    pool_out = d["pool"] if in_place else _i32(np.zeros(8))
    lens_out = d["lens"] if in_place else _i32(np.full(len(lens), -3))
    q_start = _i32(np.full(len(lens) + 1, -3))
    slots, pos = _i32(np.full(t_cap + offset + 5, -33)), _i32(np.full(t_cap + offset + 5, -33))
    assert rt.lib.sh_cuda_kv_tables(_p(d["lens"]), _p(d["add"]), len(lens), page, _p(d["table"]), table.shape[1],
                                    _p(d["ring"]), ring.size, _p(d["pool"]), _p(pool_out), _p(lens_out), _p(q_start),
                                    _p(slots) + 4 * offset, _p(pos) + 4 * offset, t_cap) == 0
    rt.check()
    for t in (slots, pos):      # nothing before or past the rows asked for
        assert (_np(t)[:offset] == -33).all() and (_np(t)[offset + t_cap:] == -33).all()
    cut = slice(offset, offset + t_cap)
    return (_np(d["table"]), _np(d["ring"]), _np(pool_out), _np(lens_out), _np(q_start), _np(slots)[cut], _np(pos)[cut])


CASES = {
    "one": ([0], [1], 16, 4, 3),
    "one_idle": ([5], [0], 16, 4, 3),
    "page_edges": ([15, 16, 17, 31, 32, 0, 0], [1, 1, 1, 2, 0, 16, 17], 16, 8, 20),
    "ends": ([40, 1, 0, 64, 33], [-1, 3, -1, -5, 7], 32, 6, 4),
    "all_end": ([40, 1, 300], [-1, -1, -1], 16, 19, 0),
    "ring_runs_out": ([16, 16, 10, 16, 0, 3], [1, 40, 2, 1, 0, 1], 16, 8, 2),
    "past_the_table": ([60, 10, 64], [10, 1, 1], 16, 4, 9),
}


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("name", CASES)
def test_tables_small(gpu_lib, name, in_place):
    lens, add, page, ld, spare = CASES[name]
    lens, add, table, ring, pool = _tables_case(lens, add, page, ld, spare, 3)
    total = int(np.maximum(add, 0).sum())
    for t_cap, offset in ((total + 3, 0), (max(total - 2, 0), 1), (4 * ((total + 3) // 4), 0)):
        want = D.kv_tables(lens, add, page, table, ring, pool, t_cap)
        got = _run_tables(gpu_lib, lens, add, page, table, ring, pool, t_cap, in_place, offset)
        for w, x in zip(want, got):
            np.testing.assert_array_equal(x[:3] if w is want[2] else x, w)
        assert not got[2][3:].any()


@pytest.mark.parametrize("R,page,add_hi,spare", [(257, 16, 3, 10 ** 4), (513, 64, 300, 3000), (1500, 32, 90, 700),
                                                 (8192, 128, 9, 10 ** 4)])
def test_tables_large(gpu_lib, R, page, add_hi, spare):
    """More requests than threads and several CTAs; the state in place, so that every CTA has to read it before one
    writes it."""
    rng = np.random.default_rng(R)
    lens = rng.integers(0, 700, R)
    add = rng.integers(0, add_hi, R)
    add[rng.random(R) < 0.06] = -1
    ld = -(-(700 + add_hi) // page)
    lens, add, table, ring, pool = _tables_case(lens, add, page, ld, spare, R)
    t_cap = int(np.maximum(add, 0).sum()) + 130
    want = D.kv_tables(lens, add, page, table, ring, pool, t_cap)
    for _ in range(3):
        got = _run_tables(gpu_lib, lens, add, page, table, ring, pool, t_cap, True)
        for w, x in zip(want, got):
            np.testing.assert_array_equal(x[:3] if w is want[2] else x, w)


# ---- append ------------------------------------------------------------------------------------------------------------
def _random_codes(rng, shape, fmt):
    c = rng.integers(0, 256, shape).astype(np.uint8)
    if fmt == "fp8":
        c[(c & 127) == 127] = 0x31
    else:
        c[c == 128] = 129           # the append writes -127 .. 127
    return c


def _random_scales(rng, shape, fmt):
    return (np.float32(rng.uniform(0.5, 1.5, shape) * 3 / D.QMAX[fmt]).view(np.uint32) & 0xFFFF0000).view(np.float32)


class Pool:
    """K and V pages in one allocation (strided pages), and the oracle's copy."""

    def __init__(self, pages, heads, page, dh, fmt, seed, interleaved=False):
        rng = np.random.default_rng(seed)
        self.shape, self.fmt, self.page = (pages, heads, page, dh), fmt, page
        size = heads * page * dh
        self.stride = 2 * size + 32 if interleaved else size
        self.codes = [_random_codes(rng, self.shape, fmt) for _ in range(2)]
        self.scales = [_random_scales(rng, (pages, heads), fmt) for _ in range(2)]
        gap = size if interleaved else pages * size
        host = np.full((pages * self.stride if interleaved else 2 * pages * size), 0xA5, np.uint8)
        self.at = [0, gap]
        for i in range(2):
            np.lib.stride_tricks.as_strided(host[self.at[i]:], (pages, size), (self.stride, 1))[:] = \
                self.codes[i].reshape(pages, size)
        self.raw0 = host
        self.raw = torch.from_numpy(host.copy()).to(DEV)
        self.dev_scales = [torch.from_numpy(s.copy()).to(DEV) for s in self.scales]
        self.handle = L.Kv8(_p(self.raw) + self.at[0], _p(self.raw) + self.at[1], _p(self.dev_scales[0]),
                            _p(self.dev_scales[1]), self.stride, pages, page, heads, dh, decode.FORMATS[fmt])

    def now(self, i):
        pages, heads, page, dh = self.shape
        raw = _np(self.raw)
        return np.lib.stride_tricks.as_strided(raw[self.at[i]:], self.shape, (self.stride, page * dh, dh, 1)).copy()

    def gaps_untouched(self):
        raw, mask = _np(self.raw).copy(), self.raw0.copy()
        size = int(np.prod(self.shape[1:]))
        for i in range(2):
            for a in (raw, mask):
                np.lib.stride_tricks.as_strided(a[self.at[i]:], (self.shape[0], size), (self.stride, 1))[:] = 0
        return np.array_equal(raw, mask)


def _check_append(rt, pool, k, v, slots, ldk, ldv, offset=0):
    """k, v: host fp16 [T, heads * dh]; on the device inside rows of ldk / ldv elements from an element offset."""
    T, w = k.shape
    dev = []
    for x, ld in ((k, ldk), (v, ldv)):
        buf = torch.full((T * ld + 16,), 60000.0, dtype=torch.float16, device=DEV)
        buf[offset:offset + T * ld].view(T, ld)[:, :w] = torch.from_numpy(x).to(DEV)
        dev.append(buf)
    d_slots = _i32(slots)
    want = [D.kv8_append(pool.now(i), _np(pool.dev_scales[i]), x, slots, pool.page, pool.fmt) for i, x in enumerate((k, v))]
    assert rt.lib.sh_cuda_kv8_append(pool.handle, _p(dev[0]) + 2 * offset, _p(dev[1]) + 2 * offset, T, ldk, ldv, _p(d_slots)) == 0
    rt.check()
    for i in range(2):
        np.testing.assert_array_equal(_np(pool.dev_scales[i]).astype(np.float64), want[i][1])
        got = pool.now(i)
        if pool.fmt == "fp8":     # zero has two codes
            got, ref = D.decode(got, "fp8"), D.decode(want[i][0], "fp8")
        else:
            ref = want[i][0]
        np.testing.assert_array_equal(got, ref)
    assert pool.gaps_untouched()


def _runs(spans, page):
    """Slots of (page id, first, last + 1) spans."""
    return np.concatenate([p * page + np.arange(a, b) for p, a, b in spans])


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("page,heads,dh,spans", [
    (16, 1, 64, [(2, 0, 1)]),                                          # a fresh page
    (16, 3, 128, [(2, 15, 16)]),                                       # the page's last row
    (32, 2, 64, [(5, 7, 8), (0, 0, 1), (1, 31, 32), (6, 12, 13)]),     # one token each
    (64, 2, 128, [(3, 20, 64), (4, 0, 64), (1, 0, 9), (0, 63, 64)]),   # a prompt over pages
    (128, 5, 64, [(1, 127, 128), (2, 0, 128), (0, 0, 128), (3, 0, 1), (4, 5, 90)]),
    (16, 8, 128, [(p, (3 * p) % 16, (3 * p) % 16 + 1) for p in range(40)]),
])
def test_append_matches_the_definition(gpu_lib, fmt, page, heads, dh, spans):
    rng = np.random.default_rng(page + dh)
    pool = Pool(max(p for p, _, _ in spans) + 2, heads, page, dh, fmt, 5)
    slots = _runs(spans, page)
    w = heads * dh
    for size in (0.01, 1.0, 30.0):      # smaller than, like and beyond what the scales cover
        k, v = ((rng.standard_normal((slots.size, w)) * size).astype(np.float16) for _ in range(2))
        _check_append(gpu_lib, pool, k, v, slots, w, w)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_append_many_rows_and_padding(gpu_lib, fmt):
    """A long prompt (whole pages per CTA), rows without a slot between and after, strides, odd addresses."""
    rng = np.random.default_rng(8)
    heads, dh, page = 4, 128, 16
    pool = Pool(700, heads, page, dh, fmt, 6, interleaved=True)
    order = rng.permutation(690)
    spans = [(int(p), 0 if i % 5 else 3, 16 if i % 7 else 11) for i, p in enumerate(order[:600])]
    slots = np.concatenate([[-1], _runs(spans[:199], page), [-1, -1, -5], _runs(spans[199:], page), [-1] * 37])
    w = heads * dh
    k, v = (rng.standard_normal((slots.size, w)).astype(np.float16) for _ in range(2))
    _check_append(gpu_lib, pool, k, v, slots, w + 8, w + 24)
    _check_append(gpu_lib, pool, k, v, slots, w + 3, w, offset=1)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_append_extremes(gpu_lib, fmt):
    """Zeros (scale 0, also over an older page), infinities, NaN, the smallest and the largest fp16."""
    page, heads, dh = 16, 2, 64
    pool = Pool(6, heads, page, dh, fmt, 9)
    pool.dev_scales[0][3] = 0.0
    pool.scales[0][3] = 0.0
    rows = np.zeros((5, heads * dh), np.float16)
    rows[1, 5], rows[1, 70], rows[1, 71] = np.inf, np.nan, -1.0
    rows[2, :] = np.float16(2.0 ** -24)
    rows[3, 3], rows[3, 100] = 65504.0, -65504.0
    rows[4, ::2] = -np.inf
    slots = np.array([0 * 16 + 0, 1 * 16 + 4, 2 * 16 + 0, 4 * 16 + 9, 5 * 16 + 15])
    _check_append(gpu_lib, pool, rows, rows[::-1].copy(), slots, heads * dh, heads * dh)
    _check_append(gpu_lib, pool, rows[:1], rows[:1], np.array([3 * 16 + 2]), heads * dh, heads * dh)     # 0 over scale 0
    _check_append(gpu_lib, pool, rows[3:4], rows[3:4], np.array([3 * 16 + 3]), heads * dh, heads * dh)


def test_append_wrong_slots_write_nothing_else(gpu_lib):
    """Slots past the cache and slots that do not rise are left out and reported; the rows beside them arrive."""
    page, heads, dh = 16, 2, 64
    rng = np.random.default_rng(3)
    k = rng.standard_normal((6, heads * dh)).astype(np.float16)
    for slots, kept in (([3, 3, 4, 9 * 16, 2 ** 31 - 1, 20], [0, 2, 5]), ([5 * 16 + 2, 5 * 16 + 1, 5 * 16 + 7, 0, 1, 1], [0, 2, 3, 4])):
        pool = Pool(8, heads, page, dh, "int8", 2)
        want = D.kv8_append(pool.now(0), _np(pool.dev_scales[0]), k[kept], np.array(slots)[kept], page, "int8")
        x, s = torch.from_numpy(k).to(DEV), _i32(slots)
        assert gpu_lib.lib.sh_cuda_kv8_append(pool.handle, _p(x), _p(x), 6, heads * dh, heads * dh, _p(s)) == 0
        assert gpu_lib.lib.sh_cuda_device_error() == 2
        np.testing.assert_array_equal(pool.now(0), want[0])
        np.testing.assert_array_equal(_np(pool.dev_scales[0]).astype(np.float64), want[1])


# ---- attention -----------------------------------------------------------------------------------------------------------
def _attn_tol(want, mean_abs, big, keys, H, dh, vmax):
    """Half-step roundings: the output's (2^-11, or 2^-25 below the normal range); the weights' before the second product
    (2^-11 of each, 2^-25 of the largest for those below the normal range); the exponent's error from the fp32 sum over
    dh products (at most dh + 4 roundings of the largest partial sum, numerator and denominator) and 2^-21 for exp2 and
    the logarithm of the scale; fp32 sums over the keys."""
    n = keys[:, None].astype(np.float64)
    b = np.repeat(big, dh, 1)
    eps_x = 2 * ((dh + 4) * 2.0 ** -24 * b + 8 * 2.0 ** -24 * (b + 64) + 2.0 ** -21)
    return 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + (2.0 ** -11 + eps_x + 2 * n * 2.0 ** -24) * mean_abs * 1.01 + n * 2.0 ** -25 * vmax


def _attn_case(rt, fmt, H, heads, dh, page, lens, nq, scale=None, seed=1, interleaved=False, ldq=None, ldo=None, offset=0,
               max_q=None, t_extra=2, mutate=None, stream=None):
    rng = np.random.default_rng(seed)
    lens, nq = np.asarray(lens), np.asarray(nq)
    R = lens.size
    blocks = np.maximum(-(-lens // page), 0)
    pages = int(blocks.sum()) + 3
    pool = Pool(pages, heads, page, dh, fmt, seed, interleaved)
    ids = rng.permutation(pages)
    ld = int(blocks.max()) + 1
    table = np.full((R, ld), 2 ** 30, np.int64)          # entries behind a request's blocks are not looked at
    at = 0
    for r in range(R):
        table[r, :blocks[r]] = ids[at:at + blocks[r]]
        at += blocks[r]
    if mutate:
        mutate(pool, table, lens, ids[at:])
    q_start = np.concatenate([[0], np.cumsum(nq)])
    T = int(q_start[-1])
    scale = 1 / math.sqrt(dh) if scale is None else scale
    w = H * dh
    ldq, ldo = ldq or w, ldo or w
    q = rng.standard_normal((T, w)).astype(np.float16)
    dq = torch.full(((T + t_extra) * ldq + 16,), float("nan"), dtype=torch.float16, device=DEV)
    dq[offset:offset + (T + t_extra) * ldq].view(-1, ldq)[:T, :w] = torch.from_numpy(q).to(DEV)
    do = torch.full(((T + t_extra) * ldo + 16,), 7.0, dtype=torch.float16, device=DEV)
    ws = torch.zeros(L.KV8_WS_BYTES, dtype=torch.uint8, device=DEV)
    d_table, d_lens, d_start = _i32(table), _i32(lens), _i32(q_start)
    want, mean_abs, big, keys = D.attention_kv8(q, pool.codes[0], pool.codes[1], pool.scales[0], pool.scales[1], table, lens,
                                                q_start, H, scale, fmt)
    mq = int(nq.max()) if max_q is None else max_q

    def call():
        assert rt.lib.sh_cuda_attention_kv8(_p(dq) + 2 * offset, _p(do) + 2 * offset, pool.handle, _p(d_table), ld, _p(d_lens),
                                            _p(d_start), R, T + t_extra, mq, H, ldq, ldo, scale, _p(ws), ws.numel()) == 0
    call()
    rt.check()
    raw = _np(do)
    got = raw[offset:offset + (T + t_extra) * ldo].reshape(-1, ldo)
    assert (got[T:] == 7).all() and (got[:, w:] == 7).all() and (raw[:offset] == 7).all()
    vmax = max(np.abs(D.decode(pool.codes[1], fmt) * pool.scales[1][:, :, None, None]).max(), 0.0) if lens.max() else 0.0
    err = np.abs(got[:T, :w].astype(np.float64) - want)
    tol = _attn_tol(want, mean_abs, big, keys, H, dh, vmax)
    bad = ~(err <= tol)
    assert not bad.any(), (np.argwhere(bad)[:4], err[bad][:4], tol[bad][:4])
    call()                               # the workspace is as it was before the first call
    rt.check()
    assert np.array_equal(_np(do).view(np.uint16), raw.view(np.uint16))
    return got[:T, :w]


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_attention_single_tokens_of_many_lengths(gpu_lib, fmt, dh, page):
    lens = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 200, 255, 257, 1000]
    _attn_case(gpu_lib, fmt, 8, 2, dh, page, lens, [1] * len(lens))


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("H,heads,dh", [(1, 1, 64), (5, 5, 64), (15, 5, 64), (32, 8, 128), (8, 1, 128), (24, 3, 64), (9, 1, 128),
                                        (16, 1, 64), (40, 2, 128)])
def test_attention_head_groups(gpu_lib, fmt, H, heads, dh):
    _attn_case(gpu_lib, fmt, H, heads, dh, 16, [70, 1, 300], [1, 1, 1])
    _attn_case(gpu_lib, fmt, H, heads, dh, 32, [70, 3, 300, 9], [5, 3, 2, 9])


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dh,H,heads", [(64, 4, 2), (128, 4, 1), (128, 3, 3)])
def test_attention_prompt_chunks(gpu_lib, fmt, dh, H, heads):
    """Whole prompts, chunks behind a cached prefix, single tokens and idle requests in one call."""
    _attn_case(gpu_lib, fmt, H, heads, dh, 16, [150, 200, 1, 77, 40, 33], [150, 61, 1, 0, 1, 33])
    _attn_case(gpu_lib, fmt, H, heads, dh, 64, [129, 260], [128, 65])


def test_attention_rows_without_keys(gpu_lib):
    """More new rows than tokens (a request that was put off keeps its length): the first rows have no key and give zeros; a
    request without tokens gives zeros throughout."""
    got = _attn_case(gpu_lib, "int8", 4, 2, 64, 16, [2, 0, 5], [5, 3, 1])
    assert (got[:3] == 0).all() and (got[5:8] == 0).all() and (got[3:5] != 0).any()
    got = _attn_case(gpu_lib, "fp8", 4, 1, 128, 16, [2, 0, 90], [40, 30, 70])
    assert (got[:38] == 0).all() and (got[40:70] == 0).all()


@pytest.mark.parametrize("nq", [1, 3, 40, 90])
def test_attention_strides_and_odd_addresses(gpu_lib, nq):
    for ldq, ldo, offset in ((4 * 64 + 8, 4 * 64 + 2, 0), (4 * 64 + 3, 4 * 64 + 1, 0), (4 * 64, 4 * 64, 1)):
        _attn_case(gpu_lib, "int8", 4, 2, 64, 32, [50, 140], [nq, nq], ldq=ldq, ldo=ldo, offset=offset, interleaved=True)


@pytest.mark.parametrize("max_q", [1, 4, 1000])
def test_attention_max_q_only_picks_the_kernel(gpu_lib, max_q):
    _attn_case(gpu_lib, "fp8", 8, 2, 64, 16, [100, 31, 260], [1, 31, 100], max_q=max_q)


@pytest.mark.parametrize("scale", [0.0, -0.125, 3.0])
@pytest.mark.parametrize("nq", [1, 30, 80])
def test_attention_scales_of_the_softmax(gpu_lib, scale, nq):
    _attn_case(gpu_lib, "int8", 4, 2, 64, 16, [300, 47], [nq, nq], scale=scale)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("nq", [1, 30, 80])
def test_attention_scales_far_apart(gpu_lib, fmt, nq):
    """Value scales from 2^-40 to 2^3 and zero (with codes of zero, as the append leaves them) in one request: the
    exponent carries them, so no weight leaves fp16's range."""
    def mutate(pool, table, lens, spare):
        pages, heads = pool.scales[1].shape
        e = np.random.default_rng(2).integers(-40, 4, (pages, heads))
        pool.scales[1][:] = np.ldexp(1.0, e)
        pool.scales[1][table[0, 2]] = 0.0
        pool.codes[1][table[0, 2]] = 0
        pool.scales[0][table[0, 1]] = 0.0
        for i in range(2):
            pool.dev_scales[i].copy_(torch.from_numpy(pool.scales[i]))
        raw = _np(pool.raw).copy()
        size = int(np.prod(pool.shape[1:]))
        raw[pool.at[1]:pool.at[1] + size * pages] = pool.codes[1].reshape(-1)
        pool.raw.copy_(torch.from_numpy(raw))
    _attn_case(gpu_lib, fmt, 4, 2, 64, 16, [200, 60], [nq, nq], mutate=mutate)


@pytest.mark.parametrize("nq", [1, 30, 80])
def test_attention_ignores_what_lies_behind_a_request(gpu_lib, nq):
    """NaN codes in the rows behind the last token and in free pages, NaN scales of free pages, wild table entries behind the
    request's blocks."""
    def mutate(pool, table, lens, spare):
        pages, heads, page, dh = pool.shape
        raw = _np(pool.raw).copy().reshape(2, pages, heads, page, dh)
        for r, n in enumerate(lens):
            if n % page:
                raw[:, table[r, n // page], :, n % page:] = 0x7F
        raw[:, spare] = 0xFF
        pool.raw.copy_(torch.from_numpy(raw.reshape(-1)))
        for i in range(2):
            pool.dev_scales[i][torch.from_numpy(spare).to(DEV)] = float("nan")
    _attn_case(gpu_lib, "fp8", 4, 2, 64, 32, [31, 33, 70, 1 + nq, 128], [1, nq, nq, 1 + nq, 1], mutate=mutate)


@pytest.mark.parametrize("nq", [1, 30, 80])
def test_attention_wrong_tables_and_lengths_are_reported(gpu_lib, nq):
    """A table entry outside the cache and a length past the table: the error word, no fault, other requests intact."""
    rt = gpu_lib
    pool = Pool(20, 2, 16, 64, "int8", 4)
    table = np.arange(12).reshape(3, 4)
    bad = table.copy()
    bad[0, 1], bad[0, 2] = 20, -1
    q = torch.randn((3 * nq, 256), device=DEV).half()
    start = _i32(np.arange(4) * nq)
    ws = torch.zeros(L.KV8_WS_BYTES, dtype=torch.uint8, device=DEV)

    def run(tab, lens):
        o, t, n = torch.zeros_like(q), _i32(tab), _i32(lens)
        assert rt.lib.sh_cuda_attention_kv8(_p(q), _p(o), pool.handle, _p(t), 4, _p(n), _p(start), 3, 3 * nq, nq, 4, 256, 256,
                                            0.125, _p(ws), ws.numel()) == 0
        err = rt.lib.sh_cuda_device_error()
        return _np(o), err
    good, err = run(table, [64, 50, 61])
    assert err == 0
    got, err = run(bad, [64, 50, 61])
    assert err == 2 and np.array_equal(got[nq:], good[nq:]) and np.isfinite(got).all()
    got, err = run(table, [1000, 50, 61])
    assert err == 2 and np.array_equal(got[nq:], good[nq:]) and np.isfinite(got).all()


def test_attention_pages_past_4_gib(gpu_lib):
    """Byte offsets beyond 32 bits: pages at the end of a 5 GiB pool give what the same pages at its beginning give."""
    rt, rng = gpu_lib, np.random.default_rng(1)
    heads, page, dh, H = 8, 64, 128, 16
    size = heads * page * dh
    pages = (5 << 30) // size
    pool = torch.zeros(pages * size, dtype=torch.uint8, device=DEV)
    small = torch.from_numpy(_random_codes(rng, (4, size), "int8")).to(DEV)
    pool.view(pages, size)[:4] = small
    pool.view(pages, size)[-4:] = small
    scales = torch.full((pages, heads), 0.02, device=DEV)
    h = L.Kv8(_p(pool), _p(pool), _p(scales), _p(scales), size, pages, page, heads, dh, L.SH_INT8)
    ws = torch.zeros(L.KV8_WS_BYTES, dtype=torch.uint8, device=DEV)
    for nq in (1, 20, 40):
        q = torch.from_numpy(rng.standard_normal((nq, H * dh)).astype(np.float16)).to(DEV)
        outs = []
        for first in (0, pages - 4):
            t, n, s, o = _i32(first + np.arange(4)), _i32([200]), _i32([0, nq]), torch.zeros_like(q)
            assert rt.lib.sh_cuda_attention_kv8(_p(q), _p(o), h, _p(t), 4, _p(n), _p(s), 1, nq, nq, H, H * dh, H * dh, 0.09,
                                                _p(ws), ws.numel()) == 0
            rt.check()
            outs.append(_np(o))
        assert np.abs(outs[0]).max() > 0.01
        np.testing.assert_array_equal(outs[0], outs[1])
    # and the append reaches them
    x = torch.from_numpy(rng.standard_normal((1, heads * dh)).astype(np.float16)).to(DEV)
    got = []
    for p in (1, pages - 1):
        pool.view(pages, size)[p] = 0
        s = _i32([p * page + 5])
        assert rt.lib.sh_cuda_kv8_append(h, _p(x), _p(x), 1, heads * dh, heads * dh, _p(s)) == 0
        rt.check()
        got.append(pool.view(pages, size)[p].cpu())
    assert torch.equal(got[0], got[1]) and got[0].any()


def test_attention_many_requests_and_one_long(gpu_lib):
    """More requests than the first scan's threads, most of them idle, beside one whose tokens span the whole grid."""
    lens = np.full(300, 5)
    nq = (np.arange(300) % 3 == 0).astype(int)
    lens[151], nq[151] = 5000, 1
    _attn_case(gpu_lib, "int8", 4, 1, 64, 64, lens, nq)


@pytest.mark.parametrize("fmt,dh,scale", [("int8", 64, None), ("fp8", 128, -0.2), ("int8", 128, 2.0)])
def test_attention_chunks_behind_long_prefixes(gpu_lib, fmt, dh, scale):
    """Chunks whose keys span many CTAs, with tiles of rows that end inside a request, beside many short ones."""
    lens, nq = np.full(40, 100), np.where(np.arange(40) % 2, 70, 1)
    lens[7], nq[7] = 9000, 65
    lens[20], nq[20] = 4001, 130
    _attn_case(gpu_lib, fmt, 2, 1, dh, 32, lens, nq, scale=scale)


@pytest.mark.parametrize("nq", [1, 12, 80])
def test_attention_infinite_and_nan_queries_stay_in_their_rows(gpu_lib, nq):
    """A row of Q with an infinity or a NaN gives NaN for its own head and leaves the others' bits as they were."""
    rt = gpu_lib
    pool = Pool(8, 2, 32, 64, "int8", 4)
    q = torch.randn((2 * nq, 256), device=DEV, generator=torch.Generator(DEV).manual_seed(1)).half()
    start, table, lens = _i32([0, nq, 2 * nq]), _i32([[0, 1, 2, 3], [4, 5, 6, 7]]), _i32([100, 128])
    ws = torch.zeros(L.KV8_WS_BYTES, dtype=torch.uint8, device=DEV)

    def run(x):
        o = torch.zeros_like(x)
        assert rt.lib.sh_cuda_attention_kv8(_p(x), _p(o), pool.handle, _p(table), 4, _p(lens), _p(start), 2, 2 * nq, nq, 4, 256, 256,
                                            0.125, _p(ws), ws.numel()) == 0
        rt.check()
        return _np(o).view(np.uint16).reshape(2 * nq, 4, 64), _np(o).reshape(2 * nq, 4, 64)
    good, _ = run(q)
    for v in (float("inf"), float("nan")):
        x = q.clone()
        x[nq, 64 + 9] = v
        bits, got = run(x)
        assert np.isnan(got[nq, 1]).all()
        rest = np.ones(good.shape[:2], bool)
        rest[nq, 1] = False
        assert np.array_equal(bits[rest], good[rest])


@pytest.mark.parametrize("max_q", [1, 12, 80])
def test_attention_idle_requests_and_fewer_rows_than_q_start(gpu_lib, max_q):
    """Nothing is written where no request has a row, nor past T when q_start goes further."""
    rt = gpu_lib
    pool = Pool(8, 2, 32, 64, "int8", 4)
    q = torch.randn((170, 256), device=DEV, generator=torch.Generator(DEV).manual_seed(2)).half()
    table, lens = _i32([[0, 1, 2, 3], [4, 5, 6, 7]]), _i32([100, 128])
    ws = torch.zeros(L.KV8_WS_BYTES, dtype=torch.uint8, device=DEV)

    def run(starts, T):
        o, s = torch.full_like(q, 7.0), _i32(starts)
        assert rt.lib.sh_cuda_attention_kv8(_p(q), _p(o), pool.handle, _p(table), 4, _p(lens), _p(s), 2, T, max_q, 4, 256, 256,
                                            0.125, _p(ws), ws.numel()) == 0
        rt.check()
        return _np(o)
    assert (run([5, 5, 5], 170) == 7).all()
    whole, cut = run([0, 80, 160], 170), run([0, 80, 160], 111)
    # both round the output and the weights by half a step (2^-11 of at most the largest value each); sums in fp32 beside that
    vmax = np.abs(D.decode(pool.codes[1], "int8") * pool.scales[1][:, :, None, None]).max()
    assert np.abs(cut[:111].astype(np.float64) - whole[:111]).max() <= 2 * 2.5 * 2.0 ** -11 * vmax
    assert (cut[111:] == 7).all() and (whole[160:] == 7).all() and (whole[:160] != 7).any(1).all()
    late = run([3, 83, 163], 170)
    assert (late[:3] == 7).all() and (late[163:] == 7).all() and (late[3:163] != 7).any(1).all()


# ---- 4-bit weights -------------------------------------------------------------------------------------------------------
def _w4_case(rt, M, N, K, group, zeros, epi=0, ldx=None, ldz=None, ldw=None, offset=0, seed=0):
    rng = np.random.default_rng(seed + M + N + K)
    ldx, ldz, ldw = ldx or K, ldz or N, ldw or (K // 2 + 15) // 16 * 16
    codes = rng.integers(0, 256, (N, ldw)).astype(np.uint8)
    scales = (rng.uniform(0.5, 1.5, (N, K // group)) * 0.02).astype(np.float16)
    zp = rng.integers(0, 16, (N, K // group)).astype(np.uint8) if zeros else None
    x = rng.standard_normal((M, K)).astype(np.float16)
    bias, res = rng.standard_normal(N).astype(np.float16), rng.standard_normal((M, N)).astype(np.float16)
    dx = torch.full((M * ldx + 16,), float("nan"), dtype=torch.float16, device=DEV)
    dx[offset:offset + M * ldx].view(M, ldx)[:, :K] = torch.from_numpy(x).to(DEV)
    dz = torch.full((M * ldz + 16,), 7.0, dtype=torch.float16, device=DEV)
    d = [torch.from_numpy(a).to(DEV) for a in (codes, scales, bias, res)]
    dzp = torch.from_numpy(zp).to(DEV) if zeros else None
    assert rt.lib.sh_cuda_gemv_w4(_p(dx) + 2 * offset, _p(d[0]), _p(d[1]), _p(dzp) if zeros else 0, _p(dz) + 2 * offset, M, N, K, ldx,
                                  ldw, ldz, group, _p(d[2]) if epi & L.EPI_BIAS else 0, _p(d[3]) if epi & L.EPI_RESIDUAL else 0,
                                  N if epi & L.EPI_RESIDUAL else 0, epi) == 0
    rt.check()
    raw = _np(dz)
    got = raw[offset:offset + M * ldz].reshape(M, ldz)
    assert (got[:, N:] == 7).all() and (raw[:offset] == 7).all() and (raw[offset + M * ldz:] == 7).all()
    W = D.w4_weights(codes, scales, zp, group, K)
    want = x.astype(np.float64) @ W
    mag = np.abs(x.astype(np.float64)) @ np.abs(W)
    if epi & L.EPI_BIAS:
        want = want + bias.astype(np.float64)
        mag = mag + np.abs(bias.astype(np.float64))
    if epi & L.EPI_RESIDUAL:
        want = want + res.astype(np.float64)
        mag = mag + np.abs(res.astype(np.float64))
    # one rounding to fp16; K products, the groups' scales and the epilogue's terms summed in fp32
    tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + (K + K // group + 16) * 2.0 ** -24 * mag
    err = np.abs(got[:, :N].astype(np.float64) - want)
    assert (err <= tol).all(), (np.argwhere(err > tol)[:4], float((err / tol).max()))
    return got[:, :N].copy()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 16, 17, 32])
def test_w4_rows(gpu_lib, M, group, zeros):
    _w4_case(gpu_lib, M, 200, 4 * group, group, zeros)
    _w4_case(gpu_lib, M, 129, 1024, group, zeros, L.EPI_BIAS | L.EPI_RESIDUAL)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("N", [1, 15, 16, 17, 33, 127, 960, 2560])
def test_w4_columns_and_depths(gpu_lib, group, N):
    for k in (1, 3, 7, 30):            # one group, odd numbers of groups, K that ends inside a step
        _w4_case(gpu_lib, 1, N, k * group, group, True, L.EPI_BIAS)
        _w4_case(gpu_lib, 5, N, k * group, group, False)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_w4_single_row_of_many_columns(gpu_lib, group, zeros):
    """Enough columns for the exact integer products: K inside a step, odd numbers of groups, a last tile that is not full."""
    for k in (1, 3, 8, 17):
        _w4_case(gpu_lib, 1, 7201, k * group, group, zeros, L.EPI_RESIDUAL)
    _w4_case(gpu_lib, 1, 7200, 2048, group, zeros, L.EPI_BIAS, ldx=2055, offset=1)


@pytest.mark.parametrize("M", [17, 25, 32])
@pytest.mark.parametrize("K,N", [(256, 50), (1024, 600), (1568, 5000), (2048, 333), (4096, 1000)])
def test_w4_up_to_32_rows(gpu_lib, M, K, N):
    """In one pass and in pieces, K in one and in more parts, residual and bias of the upper rows."""
    _w4_case(gpu_lib, M, N, K, 32, True, L.EPI_BIAS | L.EPI_RESIDUAL, ldx=K + 8, ldz=N + 3)


@pytest.mark.parametrize("M", [1, 12])
def test_w4_strides_and_odd_addresses(gpu_lib, M):
    for ldx, ldz, ldw, offset in ((520, 100, 256, 0), (513, 97, 272, 0), (512, 96, 1024, 1)):
        _w4_case(gpu_lib, M, 96, 512, 64, True, L.EPI_RESIDUAL, ldx=ldx, ldz=ldz, ldw=ldw, offset=offset)


@pytest.mark.parametrize("M,K,group", [(32, 8192, 64), (32, 28672, 128), (20, 65536, 32), (3, 1 << 18, 64), (1, 28672, 32),
                                       (1, 1 << 18, 128), (2, 40960, 128)])
def test_w4_deep(gpu_lib, M, K, group):
    """X over several CTAs of a cluster, and in pieces of its rows where it does not fit beside them."""
    _w4_case(gpu_lib, M, 70, K, group, True, L.EPI_BIAS | L.EPI_RESIDUAL)


def test_w4_is_deterministic_and_exact_on_whole_numbers(gpu_lib):
    """Small whole numbers: every product and sum is exact, so each term is counted once and in its place."""
    rt, rng = gpu_lib, np.random.default_rng(5)
    for M, N, K, group in ((1, 700, 4096, 128), (1, 7300, 1056, 32), (3, 333, 2016, 32), (13, 130, 4096, 64), (32, 130, 8192, 64)):
        codes = rng.integers(0, 256, (N, K // 2)).astype(np.uint8)
        scales = rng.integers(1, 3, (N, K // group)).astype(np.float16)
        x = rng.integers(-1, 2, (M, K)).astype(np.float16) * (rng.random((M, K)) < 0.05)
        d = [torch.from_numpy(a).to(DEV) for a in (x.astype(np.float16), codes, scales)]
        z = torch.zeros((M, N), dtype=torch.float16, device=DEV)
        assert rt.lib.sh_cuda_gemv_w4(_p(d[0]), _p(d[1]), _p(d[2]), 0, _p(z), M, N, K, K, K // 2, N, group, 0, 0, 0, 0) == 0
        rt.check()
        want = x.astype(np.float64) @ D.w4_weights(codes, scales, None, group, K)
        assert np.abs(want).max() < 2048
        np.testing.assert_array_equal(_np(z).astype(np.float64), want)


@pytest.mark.parametrize("M,N,K", [(2, 64, 256), (6, 64, 256), (12, 40, 16384), (2, 40, 16384), (1, 7201, 256), (1, 7201, 1024)])
def test_w4_special_rows_stay_apart(gpu_lib, M, N, K):
    """Infinity and NaN in one row of X reach that row of Z only, as IEEE sums have them."""
    at = min(1, M - 1)
    rt = gpu_lib
    x = torch.randn((M, K), device=DEV).half()
    codes = torch.randint(0, 256, (N, K // 2), device=DEV, dtype=torch.uint8)
    scales = torch.full((N, K // 128), 0.01, dtype=torch.float16, device=DEV)

    def run(x):
        z = torch.zeros((M, N), dtype=torch.float16, device=DEV)
        assert rt.lib.sh_cuda_gemv_w4(_p(x), _p(codes), _p(scales), 0, _p(z), M, N, K, K, K // 2, N, 128, 0, 0, 0, 0) == 0
        rt.check()
        return _np(z)
    good = run(x)
    rest = [i for i in range(M) if i != at]
    W = D.w4_weights(_np(codes), _np(scales), None, 128, K)
    for specials in ({17: np.nan, 200: np.inf}, {K - 1: np.inf}, {5: -np.inf}, {5: np.inf, 9: np.inf}):
        y = x.clone()
        for k, v in specials.items():
            y[at, k] = v
        got = run(y)
        assert np.array_equal(got[rest], good[rest])
        with np.errstate(invalid="ignore"):
            want = sum(W[k] * v for k, v in specials.items())          # inf, -inf, or NaN where a weight is 0
        assert np.array_equal(np.isnan(got[at]), np.isnan(want))
        ok = ~np.isnan(want)
        assert np.array_equal(got[at][ok].astype(np.float64), want[ok])


@pytest.mark.parametrize("M,N", [(1, 90), (4, 90), (1, 7201)])
def test_w4_wide_range_of_x(gpu_lib, M, N):
    """fp16 values from the smallest to the largest in one row: small ones beside weights that cancel or skip the large."""
    rt, rng = gpu_lib, np.random.default_rng(7)
    K, group = 512, 64
    codes = rng.integers(0, 256, (N, K // 2)).astype(np.uint8)
    codes[::2, :64] = 0x88                              # zero weights below the large values
    scales = rng.uniform(0.5, 1.5, (N, K // group)).astype(np.float16) * np.float16(2.0 ** -6)
    x = np.ldexp(rng.standard_normal((M, K)), rng.integers(-24, 4, (M, K))).astype(np.float16)
    x[:, :128] = np.where(rng.random((M, 128)) < 0.5, 65504.0, -65504.0)
    x[:, 128:160] = 2.0 ** -24
    d = [torch.from_numpy(a).to(DEV) for a in (x, codes, scales)]
    z = torch.zeros((M, N), dtype=torch.float16, device=DEV)
    assert rt.lib.sh_cuda_gemv_w4(_p(d[0]), _p(d[1]), _p(d[2]), 0, _p(z), M, N, K, K, K // 2, N, group, 0, 0, 0, 0) == 0
    rt.check()
    W = D.w4_weights(codes, scales, None, group, K)
    want, mag = x.astype(np.float64) @ W, np.abs(x.astype(np.float64)) @ np.abs(W)
    tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + (K + K // group + 16) * 2.0 ** -24 * mag
    got = _np(z).astype(np.float64)
    over = np.abs(want) >= 65520
    assert np.all(np.isinf(got[np.abs(want) > 65600]))
    assert (np.abs(got - want)[~over] <= tol[~over]).all()


# ---- together ------------------------------------------------------------------------------------------------------------
def _rope_table(pos, dh):
    ang = pos[:, None] / 10000.0 ** (np.arange(dh // 2) / (dh // 2))
    return np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float16)


@pytest.mark.parametrize("fmt,captured", [("int8", False), ("fp8", True)])
def test_a_decode_loop(gpu_lib, fmt, captured):
    """Two layers of projection -> RoPE -> tables -> append -> attention -> projection over a prompt and several single
    tokens, eager or with each single-token step replayed from one CUDA graph; requests join and end on the way. Every
    operator is checked on the inputs that it had."""
    rt, lib = gpu_lib, gpu_lib.lib
    rng = np.random.default_rng(12)
    R, H, heads, dh, Dm, page, group, cap, layers = 5, 6, 2, 64, 384, 16, 64, 64, 2
    wide = (H + 2 * heads) * dh
    W = []
    for _ in range(layers):
        W.append([[t if t is None else torch.from_numpy(t).to(DEV) for t in decode.quantize_w4(
            (rng.standard_normal(s) / math.sqrt(s[0])).astype(np.float32), group)] for s in ((Dm, wide), (H * dh, Dm))])
    cache = decode.KvCache(rt, layers, heads, dh, page, 24, R, 6, fmt, cap)
    x = [torch.zeros((cap, Dm), dtype=torch.float16, device=DEV) for _ in range(layers + 1)]
    qkv = [torch.zeros((cap, wide), dtype=torch.float16, device=DEV) for _ in range(layers)]
    rot = [torch.zeros_like(t) for t in qkv]
    att = [torch.zeros((cap, H * dh), dtype=torch.float16, device=DEV) for _ in range(layers)]
    tab = torch.zeros((cap, dh), dtype=torch.float16, device=DEV)
    all_tab = torch.from_numpy(_rope_table(np.arange(200.0), dh)).to(DEV)
    add = _i32(np.zeros(R))

    def w4(src, w, dst, T, K, N, res=None):
        for a in range(0, T, 32):
            m = min(32, T - a)
            assert lib.sh_cuda_gemv_w4(_p(src) + 2 * a * K, _p(w[0]), _p(w[1]), _p(w[2]), _p(dst) + 2 * a * N, m, N, K, K,
                                       w[0].shape[1], N, group, 0, _p(res) + 2 * a * N if res is not None else 0, N,
                                       L.EPI_RESIDUAL if res is not None else 0) == 0

    def step(T, max_q):
        cache.step(add)
        torch.index_select(all_tab, 0, cache.pos[:cap].long(), out=tab)
        for i in range(layers):
            w4(x[i], W[i][0], qkv[i], T, Dm, wide)
            rot[i].copy_(qkv[i])
            lib.sh_rope(_p(rot[i]), _p(rot[i]), _p(tab), T, (H + heads) * dh, wide, dh, dh, A)
            k = _p(rot[i]) + 2 * H * dh
            cache.append(i, k, k + 2 * heads * dh, wide, wide, T)
            cache.attend(i, _p(rot[i]), _p(att[i]), T, H, wide, H * dh, 0.125, max_q)
            w4(att[i], W[i][1], x[i + 1], T, H * dh, Dm, x[i])

    def snapshot():
        return {"codes": _np(cache.codes).copy(), "scales": _np(cache.scales).copy(), "table": _np(cache.table).copy(),
                "ring": _np(cache.ring).copy(), "pool": _np(cache.pool).copy(), "lens": _np(cache.lens).copy()}

    def check(before, adds, T):
        torch.cuda.synchronize()
        rt.check()
        want = D.kv_tables(before["lens"], adds, page, before["table"], before["ring"], before["pool"], cap)
        for w, got in zip(want, (cache.table, cache.ring, cache.pool[:3], cache.lens, cache.q_start, cache.slots, cache.pos)):
            np.testing.assert_array_equal(_np(got), w)
        slots, lens, q_start = want[5][:T], want[3], want[4]
        total = int(q_start[-1])
        for i in range(layers):
            xin, q_, r_, a_, out = (_np(t)[:T].astype(np.float64) for t in (x[i], qkv[i], rot[i], att[i], x[i + 1]))
            Wq, Wo = ([_np(t) if t is not None else None for t in w] for w in W[i])
            mats = [D.w4_weights(w[0], w[1], w[2], group, K) for w, K in ((Wq, Dm), (Wo, H * dh))]
            for src, mat, got, add_ in ((xin, mats[0], q_, 0.0), (a_, mats[1], out, xin)):
                ref, mag = src @ mat + add_, np.abs(src) @ np.abs(mat) + np.abs(add_)
                assert (np.abs(got - ref) <= 2.0 ** -11 * np.abs(ref) + 2.0 ** -25 + (Dm + 22) * 2.0 ** -24 * mag)[:total].all()
            rope = llm.rope(q_[:, :(H + heads) * dh], _np(tab)[:T], dh, rounding=False)
            assert (np.abs(rope - r_[:, :(H + heads) * dh]) <= 2.0 ** -10 * np.abs(rope) + 1e-5).all()
            codes = []
            for j in range(2):
                col = (H + j * heads) * dh
                c, s = D.kv8_append(before["codes"][i, j], before["scales"][i, j], _np(rot[i])[:T, col:col + heads * dh], slots,
                                    page, fmt)
                np.testing.assert_array_equal(D.decode(_np(cache.codes)[i, j], fmt), D.decode(c, fmt))
                np.testing.assert_array_equal(_np(cache.scales)[i, j].astype(np.float64), s)
                codes += [c, s]
            ref, mean_abs, big, keys = D.attention_kv8(r_[:, :H * dh], codes[0], codes[2], codes[1], codes[3], want[0], lens,
                                                       q_start, H, 0.125, fmt)
            vmax = np.abs(D.decode(codes[2], fmt) * codes[3][:, :, None, None]).max()
            tol = _attn_tol(ref, mean_abs, big, keys, H, dh, vmax)
            assert (np.abs(a_ - ref) <= tol)[:total].all()

    def feed(T):
        x[0][:T] = torch.from_numpy(rng.standard_normal((T, Dm)).astype(np.float16)).to(DEV)

    # prompts of three requests (one empty), one idle request, padded rows
    adds = np.array([20, 0, 17, 1, 0])
    add.copy_(_i32(adds))
    feed(40)
    before = snapshot()
    step(40, 20)
    check(before, adds, 40)

    graph = None
    if captured:
        keep = [t.clone() for t in (cache.codes, cache.scales, cache.table, cache.ring, cache.pool, cache.lens)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        old = rt.stream
        with torch.cuda.stream(side):
            rt.activate(side)
            add.copy_(_i32([1] * R))
            step(8, 1)                           # warm-up
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                step(8, 1)
        rt.activate(old)
        for t, k in zip((cache.codes, cache.scales, cache.table, cache.ring, cache.pool, cache.lens), keep):
            t.copy_(k)
        torch.cuda.synchronize()
    for adds in ([1, 1, 1, 1, 1], [1, 1, -1, 1, 0], [1, 1, 1, 1, 1], [-1, 1, 1, 1, 1], [1, 1, 1, -1, -1]):
        adds = np.array(adds)
        add.copy_(_i32(adds))
        feed(8)
        before = snapshot()
        if graph:
            graph.replay()
        else:
            step(8, 1)
        check(before, adds, 8)


def test_cache_refuses_other_step_tensors(gpu_lib):
    cache = decode.KvCache(gpu_lib, layers=1, heads=2, dh=64, page=16, pages=8, requests=3, blocks=2)
    for add in (torch.ones(3, dtype=torch.int64, device=DEV), _i32([1, 1]), torch.ones(3, dtype=torch.int32),
                _i32([1, 1, 1, 1, 1, 1])[::2]):
        with pytest.raises(ShCudaError):
            cache.step(add)
    with pytest.raises(ShCudaError):
        cache.append(0, 256, 256, 128, 128, 4)      # more rows than a step has
    assert _np(cache.pool).tolist()[:2] == [0, 8]


def test_two_streams_with_their_own_workspaces(gpu_lib):
    """Two captured attention graphs replayed side by side on two streams, each with its own workspace, give what one alone
    gives."""
    rt, lib = gpu_lib, gpu_lib.lib
    pool = Pool(140, 2, 32, 64, "int8", 4)
    cases, outs = [], []
    for i, (n, nq) in enumerate(((4000, 1), (400, 33))):
        q = torch.randn((nq, 512), device=DEV).half()
        keep = (q, torch.zeros_like(q), _i32(np.arange(128)), _i32([n]), _i32([0, nq]),
                torch.zeros(L.KV8_WS_BYTES, dtype=torch.uint8, device=DEV), nq)
        cases.append(keep)

    def call(c):
        assert lib.sh_cuda_attention_kv8(_p(c[0]), _p(c[1]), pool.handle, _p(c[2]), 128, _p(c[3]), _p(c[4]), 1, c[6], c[6], 8, 512, 512,
                                         0.125, _p(c[5]), c[5].numel()) == 0
    for c in cases:
        call(c)
        rt.check()
        outs.append(c[1].clone())
    old, streams, graphs = rt.stream, [torch.cuda.Stream() for _ in cases], []
    torch.cuda.synchronize()
    for c, s in zip(cases, streams):
        with torch.cuda.stream(s):
            rt.activate(s)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                for _ in range(4):
                    call(c)
            graphs.append(g)
    rt.activate(old)
    for c in cases:
        c[1].zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    rt.check()
    for c, o in zip(cases, outs):
        assert torch.equal(c[1], o)
