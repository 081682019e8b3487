"""Measured cases of the decode-step operators: page tables, the 8-bit paged K / V cache, attention over it, and
products with 4-bit weights.

Where `own` is false `run` computes an operator in its plain form (elementary torch operations in 32 bits); where it is
true it calls libsh_ops_cuda.so as a user's program does.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False
DEV = "cuda:0"
WS_BYTES = 48 << 20          # SH_CUDA_KV8_WS_BYTES
QMAX = {"int8": 127.0, "fp8": 448.0}


# ---- cases ------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of a full batch: one token each, a few requests end
        {"name": "tables_decode", "op": "tables", "R": 256, "page": 16, "ctx": 8192, "add": 1, "ended": 8},
        # admission of many prompts at once: long slot maps
        {"name": "tables_prefill", "op": "tables", "R": 1024, "page": 64, "ctx": 4096, "add": 512, "ended": 64},
        # the new token of each of 64 requests
        {"name": "append_decode_int8", "op": "append", "R": 64, "nq": 1, "ctx": 4096, "Hkv": 8, "dh": 128, "page": 16,
         "fmt": "int8"},
        # prompts entering the cache
        {"name": "append_prefill_fp8", "op": "append", "R": 4, "nq": 2048, "ctx": 4096, "Hkv": 8, "dh": 128, "page": 64,
         "fmt": "fp8"},
        # one user, short context: latency
        {"name": "attn_one_short", "op": "attn", "R": 1, "nq": 1, "ctx": 1000, "H": 32, "Hkv": 8, "dh": 128, "page": 16,
         "fmt": "int8"},
        # one user, long context: one sequence over the whole GPU
        {"name": "attn_one_long", "op": "attn", "R": 1, "nq": 1, "ctx": 131072, "H": 32, "Hkv": 8, "dh": 128, "page": 64,
         "fmt": "fp8"},
        # a served batch of requests of very different lengths
        {"name": "attn_batch", "op": "attn", "R": 64, "nq": 1, "ctx": 8192, "H": 32, "Hkv": 8, "dh": 128, "page": 16,
         "fmt": "int8"},
        # a few drafted tokens per request, narrow heads, an odd group of query heads
        {"name": "attn_draft", "op": "attn", "R": 32, "nq": 5, "ctx": 4000, "H": 15, "Hkv": 5, "dh": 64, "page": 32,
         "fmt": "fp8"},
        # prompt chunks over what is already cached
        {"name": "attn_chunk", "op": "attn", "R": 4, "nq": 512, "ctx": 8192, "H": 32, "Hkv": 8, "dh": 128, "page": 64,
         "fmt": "int8"},
        # a projection of one token
        {"name": "w4_one", "op": "w4", "M": 1, "N": 4096, "K": 4096, "group": 128, "zeros": False},
        # a wide projection of a few tokens
        {"name": "w4_batch", "op": "w4", "M": 16, "N": 14336, "K": 4096, "group": 64, "zeros": True},
        # the output layer for one token
        {"name": "w4_head", "op": "w4", "M": 1, "N": 49152, "K": 4096, "group": 128, "zeros": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["tables", "append", "attn", "attn", "attn", "w4", "w4"])
    if op == "tables":
        R = _log(rng, 1, 1500)
        return {"op": op, "R": R, "page": rng.choice([16, 32, 64, 128]), "ctx": _log(rng, 64, 8192),
                "add": _log(rng, 1, 512), "ended": rng.randint(0, R // 16)}
    fmt, page, dh = rng.choice(["int8", "fp8"]), rng.choice([16, 32, 64, 128]), rng.choice([64, 128])
    hkv = rng.choice([1, 2, 4, 5, 8])
    if op == "append":
        R = _log(rng, 1, 128)
        return {"op": op, "R": R, "nq": _log(rng, 1, max(1, 8192 // R)), "ctx": _log(rng, 64, 4096), "Hkv": hkv, "dh": dh,
                "page": page, "fmt": fmt}
    if op == "attn":
        H = hkv * rng.choice([1, 2, 3, 4, 7, 8])
        R = _log(rng, 1, 64)
        kind = rng.choice(["one", "one", "draft", "chunk"])
        if kind == "chunk":
            R, ctx = min(R, 4), _log(rng, 512, 8192)
            H = min(H, 4 * hkv)
            nq = _log(rng, 16, 512)
        else:
            ctx = _log(rng, 16, min(131072, 524288 // R))
            nq = 1 if kind == "one" else rng.randint(2, 8)
        return {"op": op, "R": R, "nq": min(nq, ctx), "ctx": ctx, "H": H, "Hkv": hkv, "dh": dh, "page": page, "fmt": fmt}
    group = rng.choice([32, 64, 128])
    K = group * max(1, _log(rng, 256, 8192) // group)
    return {"op": op, "M": rng.choice([1, 1, 2, 3, 5, 8, 16, 32]), "N": _log(rng, 100, min(40000, 190_000_000 // K)),
            "K": K, "group": group, "zeros": rng.random() < 0.5}


# ---- sizes that follow from a case -----------------------------------------------------------------------------------
def _spread(n, phase):
    """n fractions in (0, 1], the first one 1: the golden-ratio sequence, so that a case fixes its lengths."""
    return 1.0 - np.mod(np.arange(n) * 0.6180339887498949 + phase * (np.arange(n) > 0), 1.0)


def _lengths(c):
    """(context lengths after this step, new rows) of the case's requests."""
    R = c["R"]
    ctx = np.maximum(1, np.ceil(c["ctx"] * _spread(R, 0.0))).astype(np.int64)
    if c["op"] == "append":
        ctx = ctx + c["nq"]
    nq = np.maximum(1, np.ceil(c["nq"] * _spread(R, 0.37))).astype(np.int64)
    return ctx, np.minimum(nq, ctx)


def _tables_sizes(c):
    R, P = c["R"], c["page"]
    lens = np.floor(c["ctx"] * _spread(R, 0.11)).astype(np.int64)
    add = np.maximum(1, np.ceil(c["add"] * _spread(R, 0.53))).astype(np.int64)
    if c["ended"]:
        add[(np.arange(c["ended"]) * R) // c["ended"]] = -1
    have = -(-lens // P)
    need = np.where(add < 0, 0, -(-(lens + np.maximum(add, 0)) // P) - have)
    return lens, add, have, need


def work(c):
    if c["op"] == "tables":
        lens, add, have, need = _tables_sizes(c)
        T, gone = int(np.maximum(add, 0).sum()), int(have[add < 0].sum())
        # a token reads nothing of its own; each touched block's id is read once
        return {"bytes": 16 * c["R"] + 8 * T + 12 * int(need.sum()) + 8 * gone + 4 * c["R"], "flops": 0}
    if c["op"] == "append":
        ctx, nq = _lengths(c)
        T, P = int(nq.sum()), c["page"]
        pages = int((-(-ctx // P) - (ctx - nq) // P).sum())
        return {"bytes": 6 * T * c["Hkv"] * c["dh"] + 16 * pages * c["Hkv"] + 4 * T, "flops": 6 * T * c["Hkv"] * c["dh"]}
    if c["op"] == "attn":
        ctx, nq = _lengths(c)
        pages = int((-(-ctx // c["page"])).sum())
        keys = float((nq * (ctx - nq) + nq * (nq + 1) // 2).sum())
        byts = 2 * int(ctx.sum()) * c["Hkv"] * c["dh"] + 4 * int(nq.sum()) * c["H"] * c["dh"] + pages * (8 * c["Hkv"] + 4)
        return {"bytes": byts, "flops": 4.0 * c["H"] * c["dh"] * keys}
    M, N, K, g = c["M"], c["N"], c["K"], c["group"]
    return {"bytes": N * K // 2 + N * (K // g) * (3 if c["zeros"] else 2) + 2 * M * (K + N), "flops": 2.0 * M * N * K}


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _codes(shape, fmt, g):
    x = torch.randn(shape, generator=g, device=DEV)
    if fmt == "int8":
        return (x * 36.0).round().clamp(-127, 127).to(torch.int8)
    return (x * 110.0).clamp(-448, 448).to(torch.float8_e4m3fn)


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)


def prepare(c, seed):
    g = _gen(seed)
    s = {"c": dict(c)}
    if c["op"] == "tables":
        lens, add, have, need = _tables_sizes(c)
        R, P = c["R"], c["page"]
        ld = int((-(-(lens + np.maximum(add, 0)) // P)).max()) + 2
        pages = int(have.sum() + need.sum()) + 32
        perm = torch.randperm(pages, generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
        table = torch.full((R, ld), -1, dtype=torch.int32, device=DEV)
        col = torch.arange(ld, device=DEV)[None, :] < _i32(have)[:, None]
        used = int(have.sum())
        table[col] = perm[:used]
        head = int(torch.randint(0, pages, (1,), generator=g, device=DEV))
        ring = torch.full((pages,), -1, dtype=torch.int32, device=DEV)
        ring[(head + torch.arange(pages - used, device=DEV)) % pages] = perm[used:]
        T = int(np.maximum(add, 0).sum())
        cap = -(-T // 64) * 64                        # a captured step's rows are padded
        s |= {"lens": _i32(lens), "add": _i32(add), "table": table, "ring": ring, "cap": cap, "pages": pages,
              "pool": _i32([head, pages - used, 0, 0, 0, 0, 0, 0]), "pool_out": _i32([0] * 8),
              "lens_out": _i32([0] * R), "q_start": _i32([0] * (R + 1)), "slots": _i32([0] * cap), "pos": _i32([0] * cap)}
        return s
    if c["op"] == "w4":
        M, N, K = c["M"], c["N"], c["K"]
        s["x"] = torch.randn((M, K), generator=g, device=DEV).half()
        s["codes"] = torch.randint(0, 256, (N, K // 2), generator=g, device=DEV, dtype=torch.uint8)
        s["scales"] = ((torch.rand((N, K // c["group"]), generator=g, device=DEV) + 0.5) * (0.3 / math.sqrt(K))).half()
        s["zeros"] = torch.randint(5, 11, (N, K // c["group"]), generator=g, device=DEV, dtype=torch.uint8) if c["zeros"] else None
        s["res"] = torch.randn((M, N), generator=g, device=DEV).half()
        s["z"] = torch.zeros((M, N), dtype=torch.float16, device=DEV)
        return s
    ctx, nq = _lengths(c)
    R, P, Hkv, dh = c["R"], c["page"], c["Hkv"], c["dh"]
    blocks = -(-ctx // P)
    used = int(blocks.sum())
    pages = used + max(8, used // 16)
    perm = torch.randperm(pages, generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
    ld = int(blocks.max())
    table = torch.zeros((R, ld), dtype=torch.int32, device=DEV)
    table[torch.arange(ld, device=DEV)[None, :] < _i32(blocks)[:, None]] = perm[:used]
    T = int(nq.sum())
    step = 3.0 / QMAX[c["fmt"]]
    s |= {"T": T, "table": table, "lens": _i32(ctx), "q_start": _i32(np.concatenate([[0], np.cumsum(nq)])), "pages": pages,
          "max_q": int(nq.max()), "k": _codes((pages, Hkv, P, dh), c["fmt"], g), "v": _codes((pages, Hkv, P, dh), c["fmt"], g)}
    # scales as the append writes them: 8 significant bits
    for n in ("k_scale", "v_scale"):
        s[n] = ((torch.rand((pages, Hkv), generator=g, device=DEV) + 0.5) * step).to(torch.bfloat16).float()
    if c["op"] == "append":
        H = 4 * Hkv
        s["qkv"] = torch.randn((T, (H + 2 * Hkv) * dh), generator=g, device=DEV).half()      # one packed projection
        r = torch.repeat_interleave(torch.arange(R, device=DEV), _i32(nq).long())
        p = _i32(ctx - nq).long()[r] + torch.arange(T, device=DEV) - s["q_start"].long()[r]
        s["slots"] = (table[r, p // P].long() * P + p % P).int()
        return s
    s["q"] = torch.randn((T, c["H"] * dh), generator=g, device=DEV).half()
    s["o"] = torch.zeros((T, c["H"] * dh), dtype=torch.float16, device=DEV)
    s["ws"] = torch.zeros(WS_BYTES, dtype=torch.uint8, device=DEV)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------------
def _plain_tables(s):
    c = s["c"]
    P, pages = c["page"], s["pages"]
    lens, add, table = s["lens"].long(), s["add"].long(), s["table"]
    ld = table.shape[1]
    head, count = s["pool"][0].long(), s["pool"][1].long()
    ended, n = add < 0, add.clamp(min=0)
    have = (lens + P - 1) // P
    total_blocks = (lens + n + P - 1) // P
    long = total_blocks > ld
    need = torch.where(long | ended, 0, total_blocks - have)
    cum = need.cumsum(0)
    served = ~ended & ~long & ((need == 0) | (cum <= count))
    s["lens_out"].copy_(torch.where(ended, 0, torch.where(served, lens + n, lens)))
    ends = n.cumsum(0)
    s["q_start"][0] = 0
    s["q_start"][1:] = ends
    i = torch.arange(s["cap"], device=DEV)
    r = torch.searchsorted(ends, i, right=True).clamp(max=lens.numel() - 1)
    live = i < ends[-1]
    p = torch.where(live, lens[r] + i - (ends - n)[r], 0)
    b = p // P
    new = s["ring"][(head + (cum - need)[r] + b - have[r]).clamp(min=0) % pages]
    pid = torch.where(b < have[r], table[r, b.clamp(max=ld - 1)], new)
    ok = live & served[r]
    s["slots"].copy_(torch.where(ok, pid * P + p % P, -1))
    s["pos"].copy_(p)
    fresh = ok & (b >= have[r]) & (p % P == 0)
    table[r[fresh], b[fresh]] = pid[fresh]
    gone = torch.where(ended, have.clamp(max=ld), 0)
    mask = torch.arange(ld, device=DEV)[None, :] < gone[:, None]
    back = table[mask]
    s["ring"][(head + count + torch.arange(back.numel(), device=DEV)) % pages] = back
    taken = torch.where(served, need, 0).sum()
    s["pool_out"][0] = (head + taken) % pages
    s["pool_out"][1] = count - taken + back.numel()
    s["pool_out"][2] = (~ended & ~served & (n > 0)).sum()
    return [s[k] for k in ("table", "ring", "pool_out", "lens_out", "q_start", "slots", "pos")]


def _up8(x):
    """The next fp32 value with 8 significant bits (x >= 0)."""
    return ((x.view(torch.int32) + 0xFFFF) & ~0xFFFF).view(torch.float32)


def _encode(y, fmt):
    return y.round().clamp(-127, 127).to(torch.int8) if fmt == "int8" else y.clamp(-448, 448).to(torch.float8_e4m3fn)


def _plain_append_one(x, codes, scale, slots, fmt, P):
    T, (pages, Hkv, _, dh) = slots.numel(), codes.shape
    x = x.float().reshape(T, Hkv, dh).nan_to_num(0.0, 65504.0, -65504.0)
    page, off = slots.long() // P, slots.long() % P
    hit, inv = torch.unique(page, return_inverse=True)
    amax = torch.zeros((hit.numel(), Hkv), device=DEV).index_reduce_(0, inv, x.abs().amax(2), "amax")
    first = torch.full((hit.numel(),), P, device=DEV, dtype=torch.int64).index_reduce_(0, inv, off, "amin")
    old = torch.where(first[:, None] > 0, scale[hit], 0.0)
    new = torch.maximum(old, _up8(amax / torch.full_like(amax, QMAX[fmt])))
    # older rows of a page whose scale grew are rounded to the new step
    vals = codes[hit].float() * old[:, :, None, None] / torch.where(new > 0, new, 1.0)[:, :, None, None]
    older = (torch.arange(P, device=DEV)[None, :] < first[:, None])[:, None, :, None] & (new > old)[:, :, None, None]
    raw = codes.view(torch.uint8)
    raw[hit] = torch.where(older, _encode(vals, fmt).view(torch.uint8), raw[hit])
    s_tok = new[inv][:, :, None]
    raw[page, :, off] = _encode(torch.where(s_tok > 0, x / torch.where(s_tok > 0, s_tok, 1.0), 0.0), fmt).view(torch.uint8)
    scale[hit] = new


def _plain_append(s):
    c = s["c"]
    w = c["Hkv"] * c["dh"]
    k, v = s["qkv"][:, 4 * w:5 * w], s["qkv"][:, 5 * w:]
    _plain_append_one(k, s["k"], s["k_scale"], s["slots"], c["fmt"], c["page"])
    _plain_append_one(v, s["v"], s["v_scale"], s["slots"], c["fmt"], c["page"])
    return [s[n] for n in ("k", "v", "k_scale", "v_scale")]


def _plain_attn(s):
    c = s["c"]
    R, H, Hkv, dh, nq = c["R"], c["H"], c["Hkv"], c["dh"], s["max_q"]
    G = H // Hkv
    t = s["table"].long()
    L = t.shape[1] * c["page"]

    def rows(codes, scale):      # [R, Hkv, L, dh]
        x = codes[t].float() * scale[t][:, :, :, None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(R, Hkv, L, dh)

    start, lens = s["q_start"].long(), s["lens"].long()
    n = start[1:] - start[:-1]
    i = torch.arange(nq, device=DEV)
    at = (start[:-1, None] + i[None, :]).clamp(max=s["T"] - 1)
    q = s["q"].float()[at].reshape(R, nq, Hkv, G, dh).permute(0, 2, 3, 1, 4).reshape(R, Hkv, G * nq, dh)
    x = torch.matmul(q, rows(s["k"], s["k_scale"]).transpose(2, 3)) * (1.0 / math.sqrt(dh))
    last = (lens - n)[:, None] + i[None, :]                                             # [R, nq]
    keep = torch.arange(L, device=DEV)[None, None, :] <= last.clamp(max=L - 1)[:, :, None]
    x = x.reshape(R, Hkv, G, nq, L).masked_fill_(~keep[:, None, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    v = rows(s["v"], s["v_scale"])
    # rows past a request's end can hold anything
    v = torch.where((torch.arange(L, device=DEV)[None, :] < lens[:, None])[:, None, :, None], v, 0.0)
    o = torch.matmul(p.reshape(R, Hkv, G * nq, L), v).reshape(R, Hkv, G, nq, dh)
    o = o.permute(0, 3, 1, 2, 4).reshape(R, nq, H * dh)
    s["o"].copy_(o[i[None, :] < n[:, None]])
    return s["o"]


def _plain_w4(s):
    c = s["c"]
    M, N, K, g = c["M"], c["N"], c["K"], c["group"]
    u = s["codes"]
    w = torch.stack([u & 15, u >> 4], 2).reshape(N, K // g, g).float()
    w = (w - (8.0 if s["zeros"] is None else s["zeros"].float()[:, :, None])) * s["scales"].float()[:, :, None]
    z = torch.matmul(s["x"].float(), w.reshape(N, K).t()) + s["res"].float()
    s["z"].copy_(z)
    return s["z"]


# ---- the framework's calls ------------------------------------------------------------------------------------------------
def _lib():
    import sys
    if "softhier-mlir_b200" not in sys.path:
        sys.path.insert(0, "softhier-mlir_b200")
    from softhier_cuda import lib as L
    lib = L.load()
    lib.sh_cuda_set_stream(torch.cuda.current_stream().cuda_stream)
    return L, lib


def _handle(s, L):
    """The cache's descriptor, which a program keeps beside its tensors."""
    if "handle" not in s:
        c = s["c"]
        s["handle"] = L.Kv8(s["k"].data_ptr(), s["v"].data_ptr(), s["k_scale"].data_ptr(), s["v_scale"].data_ptr(),
                            c["Hkv"] * c["page"] * c["dh"], s["pages"], c["page"], c["Hkv"], c["dh"],
                            L.SH_INT8 if c["fmt"] == "int8" else L.SH_FP8)
    return s["handle"]


def _must(rc):
    if rc:
        raise RuntimeError(f"libsh_ops_cuda returned {rc}")


def _own(s):
    L, lib = _lib()
    c, p = s["c"], torch.Tensor.data_ptr
    if c["op"] == "tables":
        _must(lib.sh_cuda_kv_tables(p(s["lens"]), p(s["add"]), c["R"], c["page"], p(s["table"]), s["table"].shape[1],
                                    p(s["ring"]), s["pages"], p(s["pool"]), p(s["pool_out"]), p(s["lens_out"]),
                                    p(s["q_start"]), p(s["slots"]), p(s["pos"]), s["cap"]))
        return [s[k] for k in ("table", "ring", "pool_out", "lens_out", "q_start", "slots", "pos")]
    if c["op"] == "append":
        w, ld = c["Hkv"] * c["dh"], s["qkv"].shape[1]
        k = p(s["qkv"]) + 8 * w
        _must(lib.sh_cuda_kv8_append(_handle(s, L), k, k + 2 * w, s["T"], ld, ld, p(s["slots"])))
        return [s[n] for n in ("k", "v", "k_scale", "v_scale")]
    if c["op"] == "attn":
        ld = c["H"] * c["dh"]
        _must(lib.sh_cuda_attention_kv8(p(s["q"]), p(s["o"]), _handle(s, L), p(s["table"]), s["table"].shape[1], p(s["lens"]),
                                        p(s["q_start"]), c["R"], s["T"], s["max_q"], c["H"], ld, ld,
                                        1.0 / math.sqrt(c["dh"]), p(s["ws"]), WS_BYTES))
        return s["o"]
    M, N, K = c["M"], c["N"], c["K"]
    zeros = 0 if s["zeros"] is None else p(s["zeros"])
    _must(lib.sh_cuda_gemv_w4(p(s["x"]), p(s["codes"]), p(s["scales"]), zeros, p(s["z"]), M, N, K, K, K // 2, N, c["group"],
                              0, p(s["res"]), N, L.EPI_RESIDUAL))
    return s["z"]


def run(state):
    if own:
        return _own(state)
    return {"tables": _plain_tables, "append": _plain_append, "attn": _plain_attn, "w4": _plain_w4}[state["c"]["op"]](state)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------
def _e4m3(y):
    """y rounded to the nearest e4m3 value, ties to the even one."""
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -40))), -6) - 3)
    return np.rint(y / step) * step


def _exact_append(s):
    c, P = s["c"], s["c"]["page"]
    w = c["Hkv"] * c["dh"]
    slots = s["slots"].cpu().numpy().astype(np.int64)
    runs, at = [], 0
    while at < slots.size:                 # tokens of one page follow one another
        end = at
        while end < slots.size and slots[end] // P == slots[at] // P:
            end += 1
        runs.append((at, end, int(slots[at] // P), int(slots[at] % P)))
        at = end
    out = []
    for n, col in (("k", 4 * w), ("v", 5 * w)):
        x = s["qkv"][:, col:col + w].double().cpu().numpy().reshape(-1, c["Hkv"], c["dh"])
        val, sc = s[n].double().cpu().numpy(), s[n + "_scale"].double().cpu().numpy()
        rnd = np.rint if c["fmt"] == "int8" else _e4m3
        for a, e, page, off in runs:
            m, ex = np.frexp(np.abs(x[a:e]).max((0, 2)) / QMAX[c["fmt"]])
            need = np.ldexp(np.ceil(m * 256), ex - 8)
            old = sc[page] if off else np.zeros(c["Hkv"])
            new = np.maximum(old, need)
            d = np.where(new > 0, new, 1.0)[:, None, None]
            if off:
                val[page, :, :off] = np.where((new > old)[:, None, None], rnd(val[page, :, :off] * old[:, None, None] / d),
                                              val[page, :, :off])
            val[page, :, off:off + e - a] = rnd(x[a:e].transpose(1, 0, 2) / d)
            sc[page] = new
        out.append((val, sc))
    (k, ks), (v, vs) = out
    return [None, None, ks, vs] if c["fmt"] == "int8" else [k, v, ks, vs]


def _exact_attn(s):
    c = s["c"]
    H, Hkv, dh, P = c["H"], c["Hkv"], c["dh"], c["page"]
    G, start, lens = H // Hkv, s["q_start"].tolist(), s["lens"].tolist()
    out = torch.zeros((s["T"], H * dh), dtype=torch.float64, device=DEV)
    for r in range(c["R"]):
        a, e, n = start[r], start[r + 1], lens[r]
        ids = s["table"][r, :-(-n // P)].long()
        for h in range(Hkv):
            k = (s["k"][ids, h].double() * s["k_scale"][ids, h].double()[:, None, None]).reshape(-1, dh)[:n]
            v = (s["v"][ids, h].double() * s["v_scale"][ids, h].double()[:, None, None]).reshape(-1, dh)[:n]
            q = s["q"][a:e].double().reshape(e - a, H, dh)[:, h * G:(h + 1) * G].reshape(-1, dh)
            x = q @ k.t() / math.sqrt(dh)
            last = (n - (e - a) + torch.arange(e - a, device=DEV)).repeat_interleave(G)
            x = x.masked_fill(torch.arange(n, device=DEV)[None, :] > last[:, None], -math.inf)
            out[a:e].view(e - a, H, dh)[:, h * G:(h + 1) * G] = (torch.softmax(x, 1) @ v).reshape(e - a, G, dh)
    return out.cpu().numpy()


def _exact_w4(s):
    c, g = s["c"], s["c"]["group"]
    out = torch.zeros((c["M"], c["N"]), dtype=torch.float64, device=DEV)
    x = s["x"].double()
    for n in range(0, c["N"], 4096):
        u = s["codes"][n:n + 4096].long()
        q = torch.zeros((u.shape[0], c["K"]), dtype=torch.float64, device=DEV)
        q[:, 0::2], q[:, 1::2] = (u % 16).double(), (u // 16).double()
        zero = torch.full_like(s["scales"][n:n + 4096], 8.0).double() if s["zeros"] is None else s["zeros"][n:n + 4096].double()
        q = (q - zero.repeat_interleave(g, 1)) * s["scales"][n:n + 4096].double().repeat_interleave(g, 1)
        out[:, n:n + 4096] = x @ q.t()
    return (out + s["res"].double()).cpu().numpy()


def exact(c, seed):
    if c["op"] == "tables":
        return None                       # whole numbers only
    s = prepare(c, seed)
    return {"append": _exact_append, "attn": _exact_attn, "w4": _exact_w4}[c["op"]](s)
