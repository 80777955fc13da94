"""The serving operators' host side, without a GPU: refusals of the C entry
points (each returns before any CUDA call), and the kernels' metadata
arithmetic compiled for the host."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

from eshkol_transformer_b200 import build, k1, paged, sampling

ROOT = Path(__file__).resolve().parents[1]
FAKE = 0x10000  # never dereferenced: every call here is refused


def cache(**change):
    d = dict(struct_size=C.sizeof(paged.CacheDescriptor), keys=FAKE, values=FAKE, pages=8,
             page_size=16, kv_heads=2, head_dim=64, page_stride=2048, head_stride=1024,
             token_stride=64, dtype=0, reserved=0)
    d.update(change)
    return paged.CacheDescriptor(*[d[f] for f, _ in paged.CacheDescriptor._fields_])


def batch(**change):
    d = dict(struct_size=C.sizeof(paged.BatchDescriptor), batch=2, tokens=3, table_columns=4,
             max_new=2, max_length=64, offsets=FAKE, lengths=FAKE, page_table=FAKE, status=None)
    d.update(change)
    return paged.BatchDescriptor(*[d[f] for f, _ in paged.BatchDescriptor._fields_])


def append(lib, c=None, b=None, rope=None, k=FAKE, ks=128, v=FAKE, vs=128):
    err = k1.KernelError()
    rc = lib.et_b200_paged_append_v1(C.byref(c) if c else None, C.byref(b) if b else None,
                                     C.byref(rope) if rope else None, k, ks, v, vs, None,
                                     C.byref(err))
    return rc, err


def attend(lib, c=None, b=None, rope=None, heads=4, q=FAKE, qs=256, o=FAKE, os=256, ws=FAKE,
           size=1 << 40):
    err = k1.KernelError()
    rc = lib.et_b200_paged_attention_v1(C.byref(c) if c else None, C.byref(b) if b else None,
                                        C.byref(rope) if rope else None, heads, q, qs, o, os, None,
                                        ws, size, None, C.byref(err))
    return rc, err


BAD_CACHES = [dict(struct_size=8), dict(keys=None), dict(values=None), dict(pages=0),
              dict(page_size=0), dict(kv_heads=0), dict(head_dim=4), dict(head_dim=60),
              dict(head_dim=264), dict(dtype=3), dict(keys=FAKE + 8), dict(token_stride=63),
              dict(token_stride=66), dict(head_stride=1000), dict(page_stride=2040),
              dict(page_stride=1 << 62), dict(token_stride=-64), dict(dtype=1, token_stride=68)]
BAD_BATCHES = [dict(struct_size=8), dict(batch=-1), dict(tokens=-1), dict(table_columns=0),
               dict(table_columns=1 << 40), dict(offsets=None), dict(lengths=None),
               dict(page_table=None), dict(max_new=-1), dict(max_length=-1)]


@pytest.mark.parametrize("change", BAD_CACHES, ids=str)
def test_bad_caches_are_refused(lib, change):
    for call in (append, attend):
        rc, err = call(lib, cache(**change), batch())
        assert rc != 0 and err.message, change
    assert lib.et_b200_paged_attention_workspace_bytes_v1(C.byref(cache(**change)), 4) == 0


@pytest.mark.parametrize("change", BAD_BATCHES, ids=str)
def test_bad_batches_are_refused(lib, change):
    for call in (append, attend):
        rc, err = call(lib, cache(), batch(**change))
        assert rc != 0 and err.message, change


def test_bad_arguments_are_refused(lib):
    half = paged.RopeDescriptor(FAKE, None, 10)
    empty = paged.RopeDescriptor(FAKE, FAKE, 0)
    for kw in (dict(k=None), dict(v=None), dict(ks=127), dict(vs=64), dict(k=FAKE + 2),
               dict(ks=1 << 40), dict(rope=half), dict(rope=empty)):
        assert append(lib, cache(), batch(), **kw)[0] != 0, kw
    for kw in (dict(q=None), dict(o=None), dict(qs=255), dict(os=255), dict(q=FAKE + 2),
               dict(o=FAKE + 1), dict(heads=0), dict(heads=3), dict(ws=None), dict(ws=FAKE + 16),
               dict(size=64), dict(rope=half), dict(rope=empty)):
        assert attend(lib, cache(), batch(), **kw)[0] != 0, kw
    assert append(lib, None, batch())[0] != 0 and append(lib, cache(), None)[0] != 0
    assert attend(lib, None, batch())[0] != 0 and attend(lib, cache(), None)[0] != 0


def test_empty_steps_do_nothing(lib):
    for b in (batch(tokens=0), batch(batch=0)):
        assert append(lib, cache(), b, k=None, v=None)[0] == 0
        assert attend(lib, cache(), b, q=None, o=None, ws=None, size=0)[0] == 0


def sample(lib, logits=FAKE, uniform=FAKE, ids=FAKE, **change):
    d = dict(struct_size=C.sizeof(sampling.SamplingDescriptor), rows=2, vocabulary=100,
             row_stride=100, dtype=0, reserved=0, temperature=None, top_k=None, top_p=None,
             min_p=None)
    d.update(change)
    s = sampling.SamplingDescriptor(*[d[f] for f, _ in sampling.SamplingDescriptor._fields_])
    err = k1.KernelError()
    return lib.et_b200_sample_v1(C.byref(s), logits, uniform, ids, None, None, C.byref(err)), err


def test_bad_sampling_calls_are_refused(lib):
    for kw in (dict(struct_size=8), dict(rows=-1), dict(vocabulary=0), dict(vocabulary=(1 << 22) + 1),
               dict(row_stride=99), dict(dtype=3), dict(logits=None), dict(uniform=None),
               dict(ids=None), dict(logits=FAKE + 2)):
        rc, err = sample(lib, **kw)
        assert rc != 0 and err.message, kw
    assert lib.et_b200_sample_v1(None, FAKE, FAKE, FAKE, None, None, None) != 0
    assert sample(lib, rows=0, logits=None)[0] == 0


def test_metadata_arithmetic_on_the_host(tmp_path):
    out = tmp_path / "paged_host"
    subprocess.run([build.nvcc(), *build.ARCH, "-std=c++17", "--expt-relaxed-constexpr",
                    f"-I{build.INCLUDE}", f"-I{build.CSRC}", str(ROOT / "tests" / "paged_host.cu"),
                    "-o", str(out)], check=True)
    done = subprocess.run([str(out)], capture_output=True, text=True)
    assert done.returncode == 0 and done.stdout.strip() == "ok", done.stdout
