"""Token selection on the GPU (ns_argmax_rows, ns_sample_rows).

The reference's sampler takes logits.argmax(dim=-1) for greedy requests
(nanoserve/sampler.py:24-27); `argmax_rows` is the same selection -- first
index among equal maxima, first NaN if any -- in one HIP launch per batch.
For the others it filters by temperature, top-k and top-p and draws once
(sampler.py:28-77); `sample_rows` does so, with min-p beside them, from uniform
numbers that the caller gives, without a sort and without leaving the GPU.
"""

from __future__ import annotations

import numpy as np
import torch

from . import _lib

# One slice-key workspace per (device, stream), grown on demand; graph capture
# records its pointer, so it is allocated by the warm-up call before capture.
_workspaces: dict[tuple[int, int], torch.Tensor] = {}
# Buffers a larger one replaced: a graph captured with one of them keeps its
# address (and torch recycles stream handles), so they are never freed.
_retired: list[torch.Tensor] = []


def _workspace(device: torch.device, stream: int, nbytes: int) -> torch.Tensor:
    key = (device.index if device.index is not None else torch.cuda.current_device(), stream)
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        if torch.cuda.is_current_stream_capturing():
            # A graph captured earlier with the old buffer would keep its freed
            # address; callers warm up every shape before capturing.
            raise RuntimeError(
                f"argmax_rows needs a {nbytes}-byte workspace on stream {stream:#x} during graph "
                f"capture, but has {0 if ws is None else ws.numel()} bytes: run the largest shape "
                "once on this stream before capturing")
        if ws is not None:
            _retired.append(ws)
        ws = torch.empty(max(nbytes, 1 << 16), dtype=torch.uint8, device=device)
        _workspaces[key] = ws
    return ws


@torch.inference_mode()
def argmax_rows(logits: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """[M, N] logits (f32/f16/bf16, unit element stride) -> [M] int64 indices."""
    if logits.dim() != 2:
        raise ValueError(f"logits must be [M, N], got {tuple(logits.shape)}")
    if not logits.is_cuda:
        raise ValueError("argmax_rows needs a GPU tensor (the HIP path has no CPU fallback)")
    if logits.dtype not in _lib.DTYPE_CODES:
        raise TypeError(f"unsupported dtype {logits.dtype}")
    x = logits
    esz = x.element_size()
    if x.stride(1) != 1 or (x.stride(0) * esz) % 16 != 0 or x.data_ptr() % 16 != 0:
        x = x.contiguous()
        if (x.shape[1] * esz) % 16 != 0:
            pad = -x.shape[1] % (16 // esz)
            x = torch.nn.functional.pad(x, (0, pad), value=float("-inf"))[:, :logits.shape[1]]
    M, N = logits.shape
    if out is None:
        out = torch.empty(M, dtype=torch.int64, device=x.device)
    lib = _lib.load()
    stream = torch.cuda.current_stream(x.device).cuda_stream
    ws = _workspace(x.device, stream, lib.ns_argmax_rows_workspace_size(M, N))
    rc = lib.ns_argmax_rows(out.data_ptr(), x.data_ptr(), x.stride(0), M, N, _lib.DTYPE_CODES[x.dtype],
                            ws.data_ptr(), ws.numel(), stream)
    _lib.check(rc, "ns_argmax_rows")
    return out


def _per_row(x, rows: int, dtypes: tuple, device: torch.device, name: str) -> torch.Tensor | None:
    """A per-row setting as a contiguous [M] tensor on the device (a number is every row's)."""
    if x is None:
        return None
    if not isinstance(x, torch.Tensor):
        return torch.full((rows,), x, dtype=dtypes[0], device=device)
    if x.device != device:
        raise ValueError(f"{name} is on {x.device}, expected {device}")
    if x.dim() != 1 or x.shape[0] != rows:
        raise ValueError(f"{name} must be [{rows}], got {tuple(x.shape)}")
    if x.dtype not in dtypes:
        raise TypeError(f"{name} must be one of {dtypes}, got {x.dtype}")
    return x.contiguous()


def sample_rows(logits: torch.Tensor, uniform: torch.Tensor, temperature, top_k=None, top_p=None, min_p=None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """[M, N] logits (f32/f16/bf16) and [M] float32 uniform numbers in [0, 1) -> [M] int64 tokens.

    temperature, top_p, min_p (float32) and top_k (int32 or int64) are [M]
    tensors on the logits' device, or one number for all rows.  Tokens are
    ordered by logit descending, then index ascending; every filter keeps a
    prefix of that order:

      top_k  the first top_k                     (off for a row with top_k <= 0 or >= N)
      top_p  while the probability before a token, among the first top_k, is
             below top_p; always the first       (off with top_p >= 1)
      min_p  probabilities of at least min_p times the largest (off with min_p <= 0)

    The token is the first kept one whose running probability, renormalised
    over the kept ones, exceeds the row's uniform number.  A row with a
    temperature that is not positive, with a NaN, or whose largest logit is not
    finite takes argmax_rows' token.  `out`: a contiguous int64 [M] tensor."""
    if logits.dim() != 2:
        raise ValueError(f"logits must be [M, N], got {tuple(logits.shape)}")
    if not logits.is_cuda:
        raise ValueError("sample_rows needs a GPU tensor (the HIP path has no CPU fallback)")
    if logits.dtype not in _lib.DTYPE_CODES:
        raise TypeError(f"unsupported dtype {logits.dtype}")
    M, N = logits.shape
    device = logits.device
    x = logits if logits.stride(1) == 1 and (M < 2 or logits.stride(0) >= N) else logits.contiguous()
    f32 = (torch.float32,)
    if uniform is None or temperature is None:
        raise ValueError("uniform and temperature are needed")
    u = _per_row(uniform, M, f32, device, "uniform")
    t = _per_row(temperature, M, f32, device, "temperature")
    k = _per_row(top_k, M, (torch.int64, torch.int32), device, "top_k")
    p = _per_row(top_p, M, f32, device, "top_p")
    mp = _per_row(min_p, M, f32, device, "min_p")
    if out is None:
        out = torch.empty(M, dtype=torch.int64, device=device)
    elif out.shape != (M,) or out.dtype != torch.int64 or out.device != device or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous int64 [{M}] tensor on {device}")
    if M == 0:
        return out
    lib = _lib.load()
    nbytes = lib.ns_sample_rows_workspace_size(M, N)
    ws = torch.empty(max(nbytes, 8), dtype=torch.uint8, device=device)  # this call's own
    ptr = lambda a: None if a is None else a.data_ptr()  # noqa: E731
    _lib.launch(device, "sample_rows", lib.ns_sample_rows,
                out.data_ptr(), x.data_ptr(), max(x.stride(0), N), M, N, _lib.DTYPE_CODES[x.dtype],
                u.data_ptr(), t.data_ptr(), ptr(k), k is not None and k.dtype is torch.int64, ptr(p), ptr(mp),
                ws.data_ptr(), nbytes)
    return out


class SamplerInputs:
    """Per-row settings of a step's draw: one pinned host buffer, one device
    buffer, one copy.  Rows: uniform, temperature, top_p, min_p (float32) and
    top_k (int32)."""

    def __init__(self, device: torch.device, rows: int = 64) -> None:
        self.device = device
        self._reserve(rows)

    def _reserve(self, rows: int) -> None:
        self._host = torch.zeros(5, rows, dtype=torch.float32, pin_memory=self.device.type == "cuda")
        self._np = self._host.numpy()
        self._dev = torch.zeros(5, rows, dtype=torch.float32, device=self.device)

    def stage(self, seqs, non_blocking: bool = False) -> dict:
        """sample_rows' arguments for the next token of each sequence
        (scheduling.Sequence).  With non_blocking the host buffer is still being
        read on return: a caller that stages again before the copy is done
        needs another object."""
        n = len(seqs)
        if self._host.shape[1] < n:
            self._reserve(2 * n)
        h = self._np
        p = [s.sampling for s in seqs]
        h[0, :n] = [s.uniform(len(s.output_token_ids)) for s in seqs]
        h[1, :n] = [x.temperature for x in p]
        h[2, :n] = [x.top_p for x in p]
        h[3, :n] = [x.min_p for x in p]
        h[4].view(np.int32)[:n] = [min(x.top_k, 0x7FFFFFFF) for x in p]
        self._dev.copy_(self._host, non_blocking=non_blocking)
        d = self._dev
        return dict(uniform=d[0, :n], temperature=d[1, :n], top_p=d[2, :n], min_p=d[3, :n],
                    top_k=d[4].view(torch.int32)[:n])
