"""8-bit block-scaled operators of a served linear layer, as gfx950 kernels.

The work that a language model's pod spends its time in, next to the memory and link probes of
:mod:`.hip`: ``yoda-sniffer --probe-matrix`` runs, checks and times it on idle cards
(:func:`yoda_scheduler_amd.ops.hip.matrix_check`), and a node's own programs call it on tensors:

* :func:`add_rms_norm` — ``h = x + residual``, ``y = h / sqrt(mean(h²) + eps) * weight``, y in
  e4m3 with a scale for each 128 columns of a row;
* :func:`quantize` — a matrix in e4m3 with a scale for each 1 × 128 or 128 × 128 block;
* :func:`matmul` — ``a @ b.T (+ bias)`` of two such matrices, summed in float32.

Scales are float32 (largest magnitude / 448) or powers of two in e8m0 (the least ``2**p`` with the
largest magnitude ≤ 448 · 2**p), which the matrix instructions apply by themselves. A block of
zeros has scale 1; NaN and infinities become NaN and leave their block's scale alone.

Every call runs on the current stream of its tensors' device, allocates its outputs with torch,
waits for nothing and can be captured into a graph. This is the forward path of serving: an input
that requires a gradient is refused while gradients are recorded.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch

from . import hip

BLOCK = 128
E4M3 = torch.float8_e4m3fn
E8M0 = torch.float8_e8m0fnu
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_OUT = {torch.bfloat16: 0, torch.float16: 1}
_SCALES = (torch.float32, E8M0)

_fns: Optional[tuple] = None


def _lib() -> tuple:
    global _fns
    if _fns is None:
        l = hip.lib()
        _fns = (l.yoda_fp8_norm, l.yoda_fp8_quantize, l.yoda_fp8_matmul)
    return _fns


@functools.lru_cache(maxsize=4096)
def _workspace(m: int, n: int, kb: int, pow2: bool) -> int:
    """Bytes of workspace that the product of these sizes asks for."""
    return hip.lib().yoda_fp8_matmul_workspace(m, n, kb, pow2)


def blocks(n: int) -> int:
    """Blocks of 128 that cover ``n``."""
    return -(-n // BLOCK)


def _scales(like: torch.Tensor, rows: int, kb: int, block_rows: int, dtype: torch.dtype) -> torch.Tensor:
    """Room for the scales of ``rows`` (of blocks) x ``kb`` blocks and their padding, in the kernels' layout."""
    if block_rows == 1:
        pitch = (rows + 7) // 8 * 8
        return torch.empty_strided((pitch, kb), (1, pitch), dtype=dtype, device=like.device)
    return like.new_empty((rows, (kb + 3) // 4 * 4), dtype=dtype)


class BlockMatrix:
    """``rows`` × ``cols`` values in e4m3 with a scale for each block.

    ``data``    [rows, 128 · blocks(cols)] e4m3, contiguous; the columns from ``cols`` on are zero
    ``scales``  [blocks of rows, blocks of columns], float32 or e8m0. For ``block_rows`` 1 they lie
                block by block, each block's rows padded to a multiple of 8, for 128 row by row, each
                row padded to a multiple of 4.

    The constructor takes values that exist already (a checkpoint's): unpadded ones and scales in
    the other order are laid out once, here. Padded ones must hold zeros from ``cols`` on.
    """

    __slots__ = ("data", "_room", "rows", "cols", "block_rows")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor, cols: Optional[int] = None,
                 block_rows: int = 1) -> None:
        if values.dtype != E4M3 or values.dim() != 2:
            raise TypeError(f"values: a 2-D {E4M3} tensor, not {values.dim()}-D {values.dtype}")
        if scales.dtype not in _SCALES or scales.dim() != 2:
            raise TypeError(f"scales: a 2-D float32 or {E8M0} tensor, not {scales.dim()}-D {scales.dtype}")
        if block_rows not in (1, BLOCK):
            raise ValueError(f"block_rows: 1 or {BLOCK}, not {block_rows}")
        rows, width = values.shape
        cols = width if cols is None else int(cols)
        kb = blocks(cols)
        if cols < 1 or width not in (cols, kb * BLOCK):
            raise ValueError(f"values have {width} columns: {cols} or, padded with zeros, {kb * BLOCK} are wanted")
        want = (rows if block_rows == 1 else blocks(rows), kb)
        if tuple(scales.shape) != want:
            raise ValueError(f"scales: shape {want}, not {tuple(scales.shape)}")
        if values.device != scales.device:
            raise ValueError(f"values on {values.device}, scales on {scales.device}")
        if width != kb * BLOCK:
            padded = torch.zeros(rows, kb * BLOCK, dtype=torch.uint8, device=values.device)
            padded[:, :cols] = values.view(torch.uint8)
            values = padded.view(E4M3)
        elif not values.is_contiguous():
            values = values.contiguous()
        if values.data_ptr() % 16:
            values = values.clone()
        stride = (1, -(-rows // 8) * 8) if block_rows == 1 else (-(-kb // 4) * 4, 1)
        # (a view that has the strides by chance may end before its padding)
        if scales.stride() != stride or scales.data_ptr() % 16 or (rows % 8 if block_rows == 1 else kb % 4):
            room = _scales(scales, *want, block_rows, scales.dtype)
            room[:want[0], :kb].copy_(scales)
            scales = room
        self.data, self._room, self.rows, self.cols, self.block_rows = values, scales, rows, cols, block_rows

    @classmethod
    def _new(cls, x: torch.Tensor, block_rows: int, scale_dtype: torch.dtype) -> "BlockMatrix":
        """Room for a block matrix of x's shape on its device."""
        m = cls.__new__(cls)
        rows, cols = x.shape
        kb = (cols + 127) // 128
        m.data = x.new_empty((rows, kb * BLOCK), dtype=E4M3)
        m._room = _scales(x, rows if block_rows == 1 else (rows + 127) // 128, kb, block_rows, scale_dtype)
        m.rows, m.cols, m.block_rows = rows, cols, block_rows
        return m

    @property
    def values(self) -> torch.Tensor:
        """[rows, cols] e4m3: a view without the padding."""
        return self.data if self.cols % BLOCK == 0 else self.data[:, :self.cols]

    @property
    def scales(self) -> torch.Tensor:
        """[blocks of rows, blocks of columns]: a view without the padding."""
        r, kb = self._room.shape
        if self.block_rows == 1:
            return self._room if r == self.rows else self._room[:self.rows]
        want = self.data.shape[1] // BLOCK
        return self._room if kb == want else self._room[:, :want]

    @property
    def shape(self) -> tuple[int, int]:
        return self.rows, self.cols

    @property
    def device(self) -> torch.device:
        return self.data.device

    def __repr__(self) -> str:
        return (f"BlockMatrix({self.rows}x{self.cols}, blocks {self.block_rows}x{BLOCK}, "
                f"scales {self._room.dtype}, {self.data.device})")


_stream = torch._C._cuda_getCurrentRawStream     # current_stream(device) makes an object first: 1.8 us of a call of 10


def _refuse_matrix(t: torch.Tensor, name: str, dtype: Optional[torch.dtype] = None) -> None:
    if t.dim() != 2 or t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError(f"{name}: a 2-D tensor whose columns are neighbours, not {tuple(t.shape)} "
                         f"with strides {t.stride()}")
    if t.dtype not in _TYPES or dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name}: {'bfloat16, float16 or float32' if dtype is None else dtype}, not {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} is on {t.device}: these operators run on a GPU")


def _no_grad(*tensors: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("the 8-bit operators have no backward pass: call them under torch.no_grad()")


def _scale_kind(dtype: torch.dtype) -> int:
    if dtype not in _SCALES:
        raise TypeError(f"scale_dtype: torch.float32 or {E8M0}, not {dtype}")
    return 1 if dtype is E8M0 else 0


def _failed(rc: int, what: str) -> None:
    if rc < 0:
        raise ValueError(f"{what}: sizes out of range")
    hip._check(rc, what)


def quantize(x: torch.Tensor, block_rows: int = 1, scale_dtype: torch.dtype = torch.float32) -> BlockMatrix:
    """``x`` [rows, cols] (bfloat16, float16 or float32; any row stride) in e4m3 with a scale for
    each ``block_rows`` × 128 block: 1 for activations, 128 for weights."""
    _refuse_matrix(x, "x")
    _no_grad(x)
    pow2 = _scale_kind(scale_dtype)
    if block_rows not in (1, BLOCK):
        raise ValueError(f"block_rows: 1 or {BLOCK}, not {block_rows}")
    rows, cols = x.shape
    if cols < 1:
        raise ValueError("x has no columns")
    q = BlockMatrix._new(x, block_rows, scale_dtype)
    device = x.get_device()
    rc = _lib()[1](device, _stream(device), _TYPES[x.dtype], block_rows == BLOCK, pow2, x.data_ptr(), x.stride(0),
                   q.data.data_ptr(), q._room.data_ptr(), rows, cols)
    if rc:
        _failed(rc, "fp8 quantize")
    return q


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 scale_dtype: torch.dtype = torch.float32) -> tuple[BlockMatrix, Optional[torch.Tensor]]:
    """``h = x + residual`` rounded to x's type, ``y = h / sqrt(mean(h²) + eps) * weight``.

    Returns (y in e4m3 with 1 × 128 blocks, h); h is None without a residual. ``weight`` [cols] has
    x's type or is float32; x and residual [rows, cols] may have any row stride.
    """
    _refuse_matrix(x, "x")
    rows, cols = x.shape
    if cols < 1:
        raise ValueError("x has no columns")
    if weight.shape != (cols,) or cols > 1 and weight.stride(0) != 1:
        raise ValueError(f"weight: {cols} neighbouring values, not {tuple(weight.shape)} with strides {weight.stride()}")
    if weight.dtype != x.dtype and weight.dtype != torch.float32:
        raise TypeError(f"weight: {x.dtype} or float32, not {weight.dtype}")
    if weight.device != x.device:
        raise ValueError(f"x on {x.device}, weight on {weight.device}")
    if residual is not None:
        _refuse_matrix(residual, "residual", x.dtype)
        if residual.shape != x.shape or residual.device != x.device:
            raise ValueError(f"residual: {tuple(x.shape)} on {x.device}, not {tuple(residual.shape)} on {residual.device}")
    _no_grad(x, weight, residual)
    pow2 = _scale_kind(scale_dtype)
    q = BlockMatrix._new(x, 1, scale_dtype)
    device = x.get_device()
    if residual is None:
        h, res, r_pitch, to = None, None, 0, None
    else:
        h = torch.empty_like(x) if x.is_contiguous() else x.new_empty((rows, cols))
        res, r_pitch, to = residual.data_ptr(), residual.stride(0), h.data_ptr()
    rc = _lib()[0](device, _stream(device), _TYPES[x.dtype], weight.dtype == torch.float32, pow2, x.data_ptr(),
                   x.stride(0), res, r_pitch, weight.data_ptr(), to, q.data.data_ptr(), q._room.data_ptr(), rows, cols, eps)
    if rc:
        _failed(rc, "fp8 norm")
    return q, h


def matmul(a: BlockMatrix, b: BlockMatrix, out_dtype: torch.dtype = torch.bfloat16,
           bias: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``a @ b.T (+ bias)``: a [M, K] with 1 × 128 blocks, b [N, K] with 128 × 128 blocks, both with
    scales of one kind. Products are summed in float32 and rounded once to ``out_dtype`` (bfloat16 or
    float16), the type of ``bias`` [N] too. ``out``: [M, N] to write to, with any row stride.

    The matrix instruction adds eight neighbouring products in fixed point, cutting each off at 2^-13
    of the largest, before they reach the float32 sum: about 2^-16 of a result, well below a 16-bit
    output's own rounding and short of float32's, so there is no float32 output."""
    if a.block_rows != 1 or b.block_rows != BLOCK:
        raise ValueError(f"a has blocks of {a.block_rows} row(s) and b of {b.block_rows}: 1 and {BLOCK} are wanted")
    if a.cols != b.cols:
        raise ValueError(f"a has {a.cols} columns, b {b.cols}")
    kind = a._room.dtype
    if kind != b._room.dtype:
        raise TypeError(f"a's scales are {kind}, b's {b._room.dtype}")
    device = a.data.device
    if b.data.device != device:
        raise ValueError(f"a on {device}, b on {b.data.device}")
    if not a.data.is_cuda:
        raise ValueError(f"a is on {device}: these operators run on a GPU")
    if out_dtype not in _OUT:
        raise TypeError(f"out_dtype: bfloat16 or float16, not {out_dtype}")
    m, n = a.rows, b.rows
    if bias is not None:
        if bias.dtype != out_dtype:
            raise TypeError(f"bias: {out_dtype}, not {bias.dtype}")
        if bias.shape != (n,) or n > 1 and bias.stride(0) != 1 or bias.device != device:
            raise ValueError(f"bias: {n} neighbouring values on {device}, not {tuple(bias.shape)} on {bias.device}")
        _no_grad(bias)
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype, device=device)
    else:
        _refuse_matrix(out, "out", out_dtype)
        if out.shape != (m, n) or out.device != device or m > 1 and out.stride(0) < n:
            raise ValueError(f"out: {(m, n)} on {device} with rows apart, not {tuple(out.shape)} on {out.device} "
                             f"with strides {out.stride()}")
        _no_grad(out)
    kb, pow2 = (a.cols + 127) // 128, kind is E8M0
    room = _workspace(m, n, kb, pow2)
    ws = torch.empty(room, dtype=torch.uint8, device=device) if room else None
    index = device.index
    rc = _lib()[2](index, _stream(index), _OUT[out_dtype], pow2, a.data.data_ptr(), a._room.data_ptr(),
                   b.data.data_ptr(), b._room.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr(),
                   m, n, kb, max(out.stride(0), n), (m + 7) // 8 * 8, ws.data_ptr() if room else None, room)
    if rc:
        _failed(rc, "fp8 matmul")
    return out
