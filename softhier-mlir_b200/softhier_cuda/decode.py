"""Host side of a decode step: the paged 8-bit K / V cache with its block tables, and 4-bit weights.

    cache = KvCache(rt, layers=.., heads=.., dh=.., page=.., pages=.., requests=.., blocks=.., fmt="int8")
    cache.step(add)                                  # pages, slots, positions, lengths of this step's tokens
    for layer in range(layers):
        cache.append(layer, k, v, ldk, ldv, T)       # fp16 rows of this step's tokens
        cache.attend(layer, q, o, T, H, ldq, ldo, scale, max_q)

torch holds the memory; everything computed is a call of libsh_ops_cuda.so on the library's stream. Lengths, tables and
the pool of free pages stay on the device and are updated in place, so a captured step can be replayed.
"""
from __future__ import annotations

import numpy as np
import torch

from . import lib as _lib
from .runtime import Runtime, ShCudaError

FORMATS = {"int8": _lib.SH_INT8, "fp8": _lib.SH_FP8}


class KvCache:
    """One cache for `layers` layers: they share block tables (a page id names the same page in each layer's pool)."""

    def __init__(self, rt: Runtime, layers: int, heads: int, dh: int, page: int, pages: int, requests: int, blocks: int,
                 fmt: str = "int8", t_cap: int | None = None):
        dev = f"cuda:{rt.device}"
        self.rt, self.heads, self.dh, self.page, self.pages, self.requests = rt, heads, dh, page, pages, requests
        self.blocks, self.fmt, self.t_cap = blocks, fmt, requests if t_cap is None else t_cap

        def i32(*shape):
            return torch.zeros(shape, dtype=torch.int32, device=dev)

        self.codes = torch.zeros((layers, 2, pages, heads, page, dh), dtype=torch.uint8, device=dev)
        self.scales = torch.zeros((layers, 2, pages, heads), dtype=torch.float32, device=dev)
        self.lens, self.table = i32(requests), i32(requests, blocks)
        self.ring = torch.arange(pages, dtype=torch.int32, device=dev)
        self.pool = i32(8)
        self.pool[1] = pages
        self.q_start, self.slots, self.pos = i32(requests + 1), i32(self.t_cap), i32(self.t_cap)
        self.ws = torch.zeros(_lib.KV8_WS_BYTES, dtype=torch.uint8, device=dev)
        self.handles = [
            _lib.Kv8(self.codes[i, 0].data_ptr(), self.codes[i, 1].data_ptr(), self.scales[i, 0].data_ptr(),
                     self.scales[i, 1].data_ptr(), heads * page * dh, pages, page, heads, dh, FORMATS[fmt])
            for i in range(layers)]
        torch.cuda.synchronize(rt.device)      # filled on torch's current stream, used on the library's, whichever that is

    def _call(self, fn, *args) -> None:
        """The library works on the calling thread's current device, which may be another runtime's."""
        if torch.cuda.current_device() == self.rt.device:
            rc = fn(*args)
        else:
            with torch.cuda.device(self.rt.device):
                rc = fn(*args)
        if rc:
            raise ShCudaError(f"libsh_ops_cuda error {rc}: {self.rt.lib.sh_cuda_last_error_string().decode()}")

    def step(self, add: torch.Tensor) -> None:
        """add: int32 [requests] on the device, tokens of each request in this step (< 0: it has ended)."""
        if add.dtype != torch.int32 or add.shape != self.lens.shape or add.device != self.lens.device or not add.is_contiguous():
            raise ShCudaError(f"add is not a contiguous int32 [{self.requests}] on {self.lens.device}")
        p = torch.Tensor.data_ptr
        self._call(self.rt.lib.sh_cuda_kv_tables,
                   p(self.lens), p(add), self.requests, self.page, p(self.table), self.blocks, p(self.ring), self.pages,
                   p(self.pool), p(self.pool), p(self.lens), p(self.q_start), p(self.slots), p(self.pos), self.t_cap)

    def append(self, layer: int, k: int, v: int, ldk: int, ldv: int, T: int) -> None:
        """k, v: device addresses of fp16 [T, heads * dh]."""
        if T > self.t_cap:
            raise ShCudaError(f"{T} rows in a step of at most {self.t_cap}")
        self._call(self.rt.lib.sh_cuda_kv8_append, self.handles[layer], k, v, T, ldk, ldv, self.slots.data_ptr())

    def attend(self, layer: int, q: int, o: int, T: int, H: int, ldq: int, ldo: int, scale: float, max_q: int = 1) -> None:
        """q, o: device addresses of fp16 [T, H * dh]."""
        p = torch.Tensor.data_ptr
        self._call(self.rt.lib.sh_cuda_attention_kv8,
                   q, o, self.handles[layer], p(self.table), self.blocks, p(self.lens), p(self.q_start), self.requests, T,
                   max_q, H, ldq, ldo, scale, p(self.ws), self.ws.numel())


def _w4_scales(step: np.ndarray) -> np.ndarray:
    """fp16, nearest; below fp16's normal range, where nearest may lose any part of a step, not less than the step, so that 15 of
    them still cover the group."""
    s = step.astype(np.float16)
    return np.where((s < 2.0 ** -14) & (s.astype(np.float32) < step), np.nextafter(s, np.float16(1)), s)


def quantize_w4(w: np.ndarray, group: int, symmetric: bool = False):
    """W [K, N] -> (codes uint8 [N, K / 2 padded to 16 bytes], scales fp16 [N, K / group], zeros uint8 or None) of
    sh_cuda_gemv_w4. Per output column and group: from the smallest to the largest value in 15 steps, or with `symmetric`
    from -8 to 7 steps around a zero point of 8. Done once, on the host, when weights are loaded."""
    K, N = w.shape
    if group not in (32, 64, 128) or K % group:
        raise ValueError(f"K {K} is not a multiple of a group of 32, 64 or 128 ({group})")
    x = np.ascontiguousarray(np.asarray(w, np.float32).T).reshape(N, K // group, group)
    if not np.abs(x).max(initial=0.0) <= 65504.0:
        raise ValueError("a weight is not finite or beyond fp16")
    if symmetric:
        scales = _w4_scales(np.abs(x).max(2) / np.float32(7.0))
        zeros = None
        z = np.float32(8.0)
    else:
        lo, hi = np.minimum(x.min(2), 0.0), np.maximum(x.max(2), 0.0)
        scales = _w4_scales((hi - lo) / np.float32(15.0))
        s = np.where(scales > 0, scales, 1).astype(np.float32)
        zeros = np.clip(np.rint(-lo / s), 0, 15).astype(np.uint8)
        z = zeros.astype(np.float32)[:, :, None]
    s = np.where(scales > 0, scales, 1).astype(np.float32)[:, :, None]
    q = np.clip(np.rint(x / s) + z, 0, 15).astype(np.uint8).reshape(N, K)
    codes = np.zeros((N, (K // 2 + 15) // 16 * 16), np.uint8)
    codes[:, :K // 2] = q[:, 0::2] | q[:, 1::2] << 4
    return codes, scales, zeros
