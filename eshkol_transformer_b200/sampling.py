"""Sampling tokens from logits on torch CUDA tensors (et_b200_sample_v1), the
distributions that it draws from (et_b200_probabilities_v1), and verification of
drafted tokens against them (et_b200_verify_v1)."""
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
        device, d = self._shape_of(logits, temperature, top_k, top_p, min_p)
        if uniform is None or ids is None:
            raise ValueError("uniform and ids are required")
        f32 = torch.float32
        err = k1.KernelError()
        rc = self.lib.et_b200_sample_v1(
            C.byref(d), logits.data_ptr(), self._row_values(uniform, f32, device, "uniform"),
            self._row_values(ids, torch.int64, device, "ids"),
            self._row_values(logprobs, f32, device, "logprobs"), stream_of(stream, device),
            C.byref(err))
        if rc != 0:
            _check(rc, err)

    def probabilities(self, logits, probs, temperature=None, top_k=None, top_p=None, min_p=None,
                      stream: int | None = None) -> None:
        """probs (f32 [rows, vocabulary], dense rows) receives the distributions
        that sample draws from, 0 for what the filters drop."""
        device, d = self._shape_of(logits, temperature, top_k, top_p, min_p)
        err = k1.KernelError()
        rc = self.lib.et_b200_probabilities_v1(
            C.byref(d), logits.data_ptr(), probs.data_ptr(),
            _distributions(probs, self.rows, self.vocabulary, device, "probs"),
            stream_of(stream, device), C.byref(err))
        if rc != 0:
            _check(rc, err)

    def _shape_of(self, logits, temperature, top_k, top_p, min_p):
        device = logits.get_device()
        if device < 0 or torch.cuda.current_device() != device:
            raise ValueError("the logits must be on the current CUDA device")
        if (logits.shape != (self.rows, self.vocabulary) or logits.dtype not in DTYPES or
                (logits.stride(1) != 1 and self.vocabulary != 1)):
            raise ValueError("logits must be [rows, vocabulary] in f32, f16 or bf16 with dense rows")
        f32 = torch.float32
        return device, SamplingDescriptor(
            C.sizeof(SamplingDescriptor), self.rows, self.vocabulary,
            logits.stride(0) if self.rows > 1 else self.vocabulary, DTYPES[logits.dtype], 0,
            self._row_values(temperature, f32, device, "temperature"),
            self._row_values(top_k, torch.int64, device, "top_k"),
            self._row_values(top_p, f32, device, "top_p"),
            self._row_values(min_p, f32, device, "min_p"))


def _distributions(t, rows: int, vocabulary: int, device: int, name: str) -> int:
    """Checks f32 [rows, vocabulary]; its row stride."""
    if (t.shape != (rows, vocabulary) or t.dtype is not torch.float32 or t.get_device() != device or
            (t.stride(1) != 1 and vocabulary != 1)):
        raise ValueError(f"{name} must be f32 [rows, vocabulary] with dense rows on the call's device")
    return t.stride(0) if rows > 1 else vocabulary


class VerificationDescriptor(C.Structure):
    """et_b200_verification_v1"""
    _fields_ = [("struct_size", C.c_size_t), ("batch", C.c_int64), ("tokens", C.c_int64),
                ("vocabulary", C.c_int64), ("target_stride", C.c_int64), ("draft_stride", C.c_int64),
                ("offsets", C.c_void_p), ("drafts", C.c_void_p), ("accept_uniform", C.c_void_p),
                ("draw_uniform", C.c_void_p), ("status", C.c_void_p)]


class Verifier:
    """Verifies the drafted tokens of `batch` requests, whose rows are offsets[b]
    .. offsets[b + 1] - 1 of [tokens, ...] tensors (the rules are those of
    et_b200_verify_v1)."""

    def __init__(self, batch: int, tokens: int, vocabulary: int):
        self.lib = load()
        self.batch, self.tokens, self.vocabulary = batch, tokens, vocabulary

    def verify(self, offsets, target, drafts, draft, accept_uniform, draw_uniform, ids, accepted,
               status=None, stream: int | None = None) -> None:
        """ids (i64 [tokens]) receives each request's accepted drafts, its drawn token
        and -1 behind, accepted (i64 [batch]) the number of accepted drafts.  target f32
        [tokens, vocabulary]: the target model's distributions; drafts i64 [tokens];
        draft: the distributions they were drawn from, or None for drafts made without
        chance; accept_uniform f32 [tokens], draw_uniform f32 [batch]; offsets i64
        [batch + 1]; status i32 [1] or None.  ids may be drafts.  stream: as in
        `paged`."""
        device = target.get_device()
        if device < 0 or torch.cuda.current_device() != device:
            raise ValueError("the distributions must be on the current CUDA device")

        def dense(t, count, dtype, name):
            if (t.shape != (count,) or t.dtype is not dtype or t.get_device() != device or
                    not t.is_contiguous()):
                raise ValueError(f"{name} must be a dense {dtype} [{count}] tensor on the target's device")
            return t.data_ptr()

        rows, f32, i64 = (self.tokens, self.vocabulary), torch.float32, torch.int64
        d = VerificationDescriptor(
            C.sizeof(VerificationDescriptor), self.batch, self.tokens, self.vocabulary,
            _distributions(target, *rows, device, "target"),
            _distributions(draft, *rows, device, "draft") if draft is not None else 0,
            dense(offsets, self.batch + 1, i64, "offsets"), dense(drafts, self.tokens, i64, "drafts"),
            dense(accept_uniform, self.tokens, f32, "accept_uniform"),
            dense(draw_uniform, self.batch, f32, "draw_uniform"),
            dense(status, 1, torch.int32, "status") if status is not None else None)
        err = k1.KernelError()
        rc = self.lib.et_b200_verify_v1(
            C.byref(d), target.data_ptr(), draft.data_ptr() if draft is not None else None,
            dense(ids, self.tokens, i64, "ids"), dense(accepted, self.batch, i64, "accepted"),
            stream_of(stream, device), C.byref(err))
        if rc != 0:
            _check(rc, err)
