"""Low-rank adapters of many requests beside a shared projection, on the HIP kernels of nano-gpic_amd/csrc/lora.hip. No counterpart
in the reference.

    y = fp8_linear_rows(x, W)                  the projection that all requests share (any linear's output serves)
    y = lora_rows(y, x, A, B, ids, scale)      y + scale_i (x A_i^T) B_i^T, each row by its request's adapter i

For serving: forward only. One token of a request, prompts, and both mixed in one call take the same operator; the rows may come in
any order.
"""
from typing import Optional

import torch

from . import _lib as L
from .fp8_native import _rows
from .layernorm import no_tangents
from .rows import _run, _same_device

DTYPES = {torch.bfloat16: 0, torch.float16: 2}
MAX_RANK = 128
MAX_WIDTH = 1 << 24


def _near_rows(t):
    """_rows, and a copy where the rows lie further apart than the kernels' offsets reach."""
    t, ld = _rows(t)
    return (t, ld) if ld < 1 << 24 else _rows(t.contiguous())


def _check(y, x, A, B, ids, scale):
    L.require_gpu(y, x, A, B, ids, scale)
    if (y.dim() < 2 or x.shape[:-1] != y.shape[:-1] or A.dim() != 3 or B.dim() != 3 or A.shape[0] != B.shape[0] or A.shape[0] == 0 or
            A.shape[2] != x.shape[-1] or B.shape[1] != y.shape[-1] or A.shape[1] != B.shape[2]):
        raise ValueError(f"lora_rows takes y [..., N], x [..., K], A [n, R, K] and B [n, N, R] with n > 0, got {tuple(y.shape)}, "
                         f"{tuple(x.shape)}, {tuple(A.shape)} and {tuple(B.shape)}")
    if y.dtype not in DTYPES or any(t.dtype != y.dtype for t in (x, A, B)):
        raise ValueError(f"lora_rows takes bf16 or fp16 y, x, A and B of one type, got {y.dtype}, {x.dtype}, {A.dtype} and {B.dtype}")
    n, R, K = A.shape
    N = y.shape[-1]
    if N % 8 or K % 8 or R % 8 or not 0 < N < MAX_WIDTH or not 0 < K < MAX_WIDTH or not 0 < R <= MAX_RANK:
        raise ValueError(f"lora_rows needs N, K and R multiples of 8, N and K below 2^24 and R <= {MAX_RANK}, got N = {N}, K = {K}, "
                         f"R = {R}")
    if ids.dtype not in (torch.int32, torch.int64) or (ids.shape != x.shape[:-1] and ids.shape != x.shape[:1]):
        raise ValueError(f"ids must be int32 or int64 {tuple(x.shape[:-1])}, or [{x.shape[0]}] for the batch, got {ids.dtype} "
                         f"{tuple(ids.shape)}")
    if scale is not None and (scale.dtype != torch.float32 or scale.shape != (n,)):
        raise ValueError(f"scale must be fp32 [{n}], got {scale.dtype} {tuple(scale.shape)}")
    _same_device(y.device, x=x, A=A, B=B, ids=ids, scale=scale)
    no_tangents("lora_rows", y, x, A, B, scale)


@L.step_op("gpic::lora_rows")
def lora_rows_op(y: torch.Tensor, x: torch.Tensor, A: torch.Tensor, B: torch.Tensor, ids: torch.Tensor,
                 scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """lora_rows, as an op."""
    o = L.native("lora_rows", y, y, x, A, B, ids, scale)
    if o is not None:
        return o
    _check(y, x, A, B, ids, scale)
    (n, R, K), N = A.shape, y.shape[-1]
    out = torch.empty(y.shape, dtype=y.dtype, device=y.device)
    M = out.numel() // N
    if M == 0:
        return out
    (y2, ldy), (x2, ldx) = _near_rows(y.reshape(M, N)), _near_rows(x.reshape(M, K))
    A, B, ids = L.aligned(A.contiguous()), L.aligned(B.contiguous()), ids.contiguous()
    scale = scale.contiguous() if scale is not None else None
    with L.on_device(y.device):
        nws = L.lib().gpic_fp8_lora_rows_workspace_bytes(M, N, K, R, n)
        ws = torch.empty(nws, dtype=torch.uint8, device=y.device)
        L.check(L.lib().gpic_fp8_lora_rows(
            y2.data_ptr(), ldy, x2.data_ptr(), ldx, A.data_ptr(), B.data_ptr(), L.ptr(scale), ids.data_ptr(),
            int(ids.dtype == torch.int64), M // ids.numel(), DTYPES[y.dtype], M, N, K, R, n, out.data_ptr(), ws.data_ptr(), nws,
            L.stream_ptr(y.device)), "gpic_fp8_lora_rows")
    return out


@lora_rows_op.register_fake
def _(y, x, A, B, ids, scale=None):
    return y.new_empty(y.shape)


def lora_rows(y, x, A, B, ids, scale=None):
    """y + scale_i (x A_i^T) B_i^T, a new tensor like y: y [..., N] a shared projection's output of x [..., K]; A [n, R, K] and
    B [n, N, R] the adapters' factors (a smaller rank than R: zeros), bf16 or fp16 all four; ids int32 or int64, one a row
    (x.shape[:-1]) or one a batch entry ([x.shape[0]]): i = ids of the row, and a row whose id is none of 0 .. n - 1 (-1) keeps y;
    scale [n] fp32, or None for ones. N, K and R are multiples of 8, N and K below 2^24, R <= 128. Sums are fp32 and the result is
    rounded once. What an adapter holds (an infinity, a NaN) reaches no row but its own. Forward only."""
    return _run(lora_rows_op, "lora_rows", y, y, x, A, B, ids, scale)
