"""Sampling tokens from logits on torch CUDA tensors (et_b200_sample_v1)."""
from __future__ import annotations

import ctypes as C

import torch

from . import _check, k1, load
from .paged import DTYPES, _need


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
        self.rows, self.vocabulary = rows, vocabulary
        self.descriptor = SamplingDescriptor(C.sizeof(SamplingDescriptor), rows, vocabulary)
        self._ref = C.byref(self.descriptor)

    def _row_values(self, t, dtype, device, name: str):
        if t is None:
            return None
        _need(t.shape == (self.rows,) and t.dtype is dtype and t.device == device and
              t.is_contiguous(), f"{name} must be a dense {dtype} [rows] tensor on the logits' device")
        return t.data_ptr()

    def sample(self, logits, uniform, ids, logprobs=None, temperature=None, top_k=None, top_p=None,
               min_p=None, stream: int = 0) -> None:
        """ids (i64 [rows]) and logprobs (f32 [rows], or None) receive the
        drawn tokens and their log-probabilities; uniform f32 [rows] in
        [0, 1); temperature, top_p, min_p f32 [rows], top_k i64 [rows], or
        None."""
        d, device = self.descriptor, logits.device
        _need(logits.is_cuda and torch.cuda.current_device() == device.index,
              "the logits must be on the current CUDA device")
        _need(logits.shape == (self.rows, self.vocabulary) and logits.dtype in DTYPES and
              (logits.stride(1) == 1 or self.vocabulary == 1),
              "logits must be [rows, vocabulary] in f32, f16 or bf16 with dense rows")
        d.row_stride = logits.stride(0) if self.rows > 1 else self.vocabulary
        d.dtype = DTYPES[logits.dtype]
        d.temperature = self._row_values(temperature, torch.float32, device, "temperature")
        d.top_k = self._row_values(top_k, torch.int64, device, "top_k")
        d.top_p = self._row_values(top_p, torch.float32, device, "top_p")
        d.min_p = self._row_values(min_p, torch.float32, device, "min_p")
        err = k1.KernelError()
        _need(uniform is not None and ids is not None, "uniform and ids are required")
        _check(self.lib.et_b200_sample_v1(
            self._ref, logits.data_ptr(),
            self._row_values(uniform, torch.float32, device, "uniform"),
            self._row_values(ids, torch.int64, device, "ids"),
            self._row_values(logprobs, torch.float32, device, "logprobs"), stream, C.byref(err)),
            err)
