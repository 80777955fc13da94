"""The serving operators' host side at the ends of its ranges, without a GPU."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

from eshkol_transformer_b200 import build, k1, paged, sampling
from test_serving_host import FAKE, append, attend, batch, cache, sample

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.parametrize("page", [1, 16, 64, 1 << 20])
def test_page_tables_of_nearly_2_31_keys_are_refused(lib, page):
    """Rounded up to blocks of keys, their positions would leave 32 bits."""
    pool = cache(page_size=page, head_stride=64 * page, page_stride=128 * page)
    for columns in {(2 ** 31 - 1) // page, (2 ** 31 - 4097) // page + 1}:
        if columns * page < 2 ** 31 - 4096:  # the last whole page lies below
            continue
        for call in (append, attend):
            rc, err = call(lib, pool, batch(table_columns=columns))
            assert rc != 0 and b"limits" in err.message, (page, columns)


def test_arithmetic_at_the_largest_page_table(tmp_path):
    out = tmp_path / "paged_limits"
    subprocess.run([build.nvcc(), *build.ARCH, "-std=c++17", "--expt-relaxed-constexpr",
                    f"-I{build.INCLUDE}", f"-I{build.CSRC}", str(ROOT / "tests" / "paged_limits.cu"),
                    "-o", str(out)], check=True)
    done = subprocess.run([str(out)], capture_output=True, text=True)
    assert done.returncode == 0 and done.stdout.strip() == "ok", done.stdout


def test_workspace_of_a_refused_number_of_heads(lib):
    """No workspace where the call itself is refused (65,536 query heads at most)."""
    size = lambda heads: lib.et_b200_paged_attention_workspace_bytes_v1(C.byref(cache()), heads)
    assert size(65536) > 0
    for heads in (65538, 1 << 40, 3, 0, -2):
        assert size(heads) == 0, heads
        assert attend(lib, cache(), batch(), heads=heads, qs=1 << 31, os=1 << 31)[0] != 0


def test_misaligned_arrays_are_refused(lib):
    """Arrays off their elements' alignment, which a kernel could not read."""
    refused = lambda rc, err: rc != 0 and b"aligned" in err.message
    for field, off in (("offsets", 4), ("lengths", 4), ("page_table", 2), ("status", 1)):
        for call in (append, attend):
            assert refused(*call(lib, cache(), batch(**{field: FAKE + off}))), field
    for rope in (paged.RopeDescriptor(FAKE + 2, FAKE, 10), paged.RopeDescriptor(FAKE, FAKE + 1, 10)):
        for call in (append, attend):
            assert refused(*call(lib, cache(), batch(), rope))
    err = k1.KernelError()
    rc = lib.et_b200_paged_attention_v1(C.byref(cache()), C.byref(batch()), None, 4, FAKE, 256, FAKE, 256,
                                        FAKE + 2, FAKE, 1 << 40, None, C.byref(err))
    assert refused(rc, err)
    for kw in (dict(ids=FAKE + 4), dict(uniform=FAKE + 2), dict(top_k=FAKE + 4),
               dict(temperature=FAKE + 1), dict(top_p=FAKE + 2), dict(min_p=FAKE + 3)):
        assert refused(*sample(lib, **kw)), kw
    d = sampling.SamplingDescriptor(C.sizeof(sampling.SamplingDescriptor), 2, 100, 100, 0, 0, None, None,
                                    None, None)
    assert refused(lib.et_b200_sample_v1(C.byref(d), FAKE, FAKE, FAKE, FAKE + 2, None, C.byref(err)), err)
