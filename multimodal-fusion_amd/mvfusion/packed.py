"""Rows kept in 8 bits: what a training step holds of a layer's input until its
backward pass, at a quarter (float32) or half (16-bit types) of the bytes.

A row is cut into groups of 32 neighbouring columns.  A group has one exponent
byte, a value one signed byte: ``code * 2 ** (exponent - 133)``, the exponent the
smallest with ``amax <= 127.5 * 2 ** (exponent - 133)`` for the group's largest
finite magnitude.  A finite value reads back within half a step of itself, at
most ``amax / 127.5`` (one step for the very largest numbers of the type); a value
that is not finite reads back as NaN and leaves the rest of its group alone.
Nothing here records an autograd graph.
"""
import torch

from . import _lib as L

ROW_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
GROUP = 32


class PackedRows:
    """Rows of ``pack_rows``: ``codes`` int8 [rows, C], ``exps`` uint8
    [rows, ceil(C / 32)], and the ``dtype`` they were packed from."""

    __slots__ = ("codes", "exps", "dtype")

    def __init__(self, codes, exps, dtype):
        self.codes, self.exps, self.dtype = codes, exps, dtype

    @property
    def shape(self):
        return self.codes.shape

    @property
    def device(self):
        return self.codes.device

    @property
    def nbytes(self):
        return self.codes.numel() + self.exps.numel()

    def unpack(self, dtype=None):
        """The rows as they read back, [rows, C] of ``dtype`` (default: the one they
        were packed from).  Exact in float32 and bfloat16; float16 holds what was
        packed from float16, and rounds or overflows on other rows."""
        return unpack_rows(self.codes, self.exps, self.dtype if dtype is None else dtype)

    def __repr__(self):
        return f"PackedRows(shape={tuple(self.shape)}, dtype={self.dtype}, device={self.device})"


def _check_rows(x, what):
    if not x.is_cuda:
        raise RuntimeError(f"mvfusion {what} runs on a HIP device only (there is no CPU fallback).")
    if x.dtype not in ROW_TYPES:
        raise TypeError(f"mvfusion {what} expects float32, bfloat16 or float16 rows, got {x.dtype}")


def check_codes(codes, exps, what):
    """Refuses what is not the two parts of 8-bit rows."""
    if (codes.dtype != torch.int8 or exps.dtype != torch.uint8 or codes.dim() != 2 or codes.shape[1] < 1
            or exps.shape != (codes.shape[0], (codes.shape[1] + GROUP - 1) // GROUP) or exps.device != codes.device):
        raise ValueError(f"{what} expects int8 codes [rows, C] and uint8 exps [rows, ceil(C / 32)] on one device")


def empty_codes(rows, C, device):
    """Room for the 8-bit form of [rows, C]."""
    return (torch.empty((rows, C), dtype=torch.int8, device=device),
            torch.empty((rows, (C + GROUP - 1) // GROUP), dtype=torch.uint8, device=device))


def pack_codes(x):
    """(codes, exps) of the rows [rows, C] (``pack_rows`` without the object around them)."""
    _check_rows(x, "pack_rows")
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"pack_rows expects [rows, C] with at least one column, got {tuple(x.shape)}")
    x = x.detach().contiguous()
    rows, C = x.shape
    dev = x.device
    codes, exps = empty_codes(rows, C, dev)
    if rows:
        L.launch(dev, L.load().mvf_pack_rows8, x.data_ptr(), ROW_TYPES[x.dtype], rows, C, codes.data_ptr(),
                 exps.data_ptr())
    return codes, exps


def pack_rows(x):
    """8-bit form of the rows [rows, C] of a float32, bfloat16 or float16 tensor on
    the HIP device."""
    return PackedRows(*pack_codes(x), x.dtype)


def unpack_rows(codes, exps, dtype=torch.float32):
    """The values of 8-bit rows (``PackedRows.unpack``)."""
    if not codes.is_cuda:
        raise RuntimeError("mvfusion unpack_rows runs on a HIP device only (there is no CPU fallback).")
    if dtype not in ROW_TYPES:
        raise TypeError(f"mvfusion unpack_rows gives float32, bfloat16 or float16 rows, not {dtype}")
    check_codes(codes, exps, "unpack_rows")
    codes, exps = codes.contiguous(), exps.contiguous()
    rows, C = codes.shape
    dev = codes.device
    y = torch.empty((rows, C), dtype=dtype, device=dev)
    if rows:
        L.launch(dev, L.load().mvf_unpack_rows8, codes.data_ptr(), exps.data_ptr(), rows, C, y.data_ptr(),
                 ROW_TYPES[dtype])
    return y
