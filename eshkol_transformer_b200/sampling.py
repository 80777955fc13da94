"""Sampling tokens from logits on torch CUDA tensors (et_b200_sample_v1)."""
from __future__ import annotations

import ctypes as C

import torch

from . import _check, k1, load
from .paged import DTYPES, stream_of


class SamplingDescriptor(C.Structure):
    """et_b200_sampling_v1"""
    _fields_ = [("struct_size", C.c_size_t), ("rows", C.c_int64), ("vocabulary", C.c_int64),
                ("row_stride", C.c_int64), ("dtype", C.c_uint32), ("reserved", C.c_uint32),
                ("temperature", C.c_void_p), ("top_k", C.c_void_p), ("top_p", C.c_void_p),
                ("min_p", C.c_void_p)]


class Sampler:
    """Draws one token per row of logits [rows, vocabulary] by inversion at
    given uniform numbers, after temperature, top-k, top-p and min-p (the
    order and the ties are those of et_b200_sample_v1)."""

    def __init__(self, rows: int, vocabulary: int):
        self.lib = load()
        self.rows, self.vocabulary, self._shape = rows, vocabulary, (rows,)

    def _row_values(self, t, dtype, device, name: str):
        if t is None:
            return None
        if (t.shape != self._shape or t.dtype is not dtype or t.get_device() != device or
                not t.is_contiguous()):
            raise ValueError(f"{name} must be a dense {dtype} [rows] tensor on the logits' device")
        return t.data_ptr()

    def sample(self, logits, uniform, ids, logprobs=None, temperature=None, top_k=None, top_p=None,
               min_p=None, stream: int | None = None) -> None:
        """ids (i64 [rows]) and logprobs (f32 [rows], or None) receive the
        drawn tokens and their log-probabilities; uniform f32 [rows] in
        [0, 1); temperature, top_p, min_p f32 [rows], top_k i64 [rows], or
        None.  stream: as in `paged`."""
        device = logits.get_device()
        if device < 0 or torch.cuda.current_device() != device:
            raise ValueError("the logits must be on the current CUDA device")
        if (logits.shape != (self.rows, self.vocabulary) or logits.dtype not in DTYPES or
                (logits.stride(1) != 1 and self.vocabulary != 1)):
            raise ValueError("logits must be [rows, vocabulary] in f32, f16 or bf16 with dense rows")
        if uniform is None or ids is None:
            raise ValueError("uniform and ids are required")
        f32 = torch.float32
        d = SamplingDescriptor(
            C.sizeof(SamplingDescriptor), self.rows, self.vocabulary,
            logits.stride(0) if self.rows > 1 else self.vocabulary, DTYPES[logits.dtype], 0,
            self._row_values(temperature, f32, device, "temperature"),
            self._row_values(top_k, torch.int64, device, "top_k"),
            self._row_values(top_p, f32, device, "top_p"),
            self._row_values(min_p, f32, device, "min_p"))
        err = k1.KernelError()
        rc = self.lib.et_b200_sample_v1(
            C.byref(d), logits.data_ptr(), self._row_values(uniform, f32, device, "uniform"),
            self._row_values(ids, torch.int64, device, "ids"),
            self._row_values(logprobs, f32, device, "logprobs"), stream_of(stream, device),
            C.byref(err))
        if rc != 0:
            _check(rc, err)
