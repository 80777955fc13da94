"""The 8-bit cache's and speculative decoding's host side, without a GPU: refusals of the
C entry points (each returns before any CUDA call)."""
import ctypes as C

import pytest
import torch

from cache8_f64 import e4m3_values, quantise
from eshkol_transformer_b200 import k1, paged, sampling
from test_serving_host import BAD_BATCHES, FAKE, batch


def cache(**change):
    d = dict(struct_size=C.sizeof(paged.Cache8Descriptor), keys=FAKE, values=FAKE, key_scales=FAKE,
             value_scales=FAKE, pages=8, page_size=16, kv_heads=2, head_dim=64, page_stride=2048,
             head_stride=1024, token_stride=64, scale_page_stride=32, scale_head_stride=16,
             scale_token_stride=1, dtype=0, reserved=0)
    d.update(change)
    return paged.Cache8Descriptor(*[d[f] for f, _ in paged.Cache8Descriptor._fields_])


def append(lib, c=None, b=None, rope=None, k=FAKE, ks=128, v=FAKE, vs=128):
    err = k1.KernelError()
    rc = lib.et_b200_paged_append8_v1(C.byref(c) if c else None, C.byref(b) if b else None,
                                      C.byref(rope) if rope else None, k, ks, v, vs, None, C.byref(err))
    return rc, err


def attend(lib, c=None, b=None, rope=None, heads=4, q=FAKE, qs=256, o=FAKE, os=256, lse=None, ws=FAKE,
           size=1 << 40):
    err = k1.KernelError()
    rc = lib.et_b200_paged_attention8_v1(C.byref(c) if c else None, C.byref(b) if b else None,
                                         C.byref(rope) if rope else None, heads, q, qs, o, os, lse,
                                         ws, size, None, C.byref(err))
    return rc, err


BAD_CACHES = [dict(struct_size=8), dict(keys=None), dict(values=None), dict(key_scales=None),
              dict(value_scales=None), dict(pages=0), dict(page_size=0), dict(kv_heads=0),
              dict(head_dim=8), dict(head_dim=72), dict(head_dim=272), dict(dtype=3),
              dict(keys=FAKE + 8), dict(values=FAKE + 1), dict(key_scales=FAKE + 2),
              dict(value_scales=FAKE + 1), dict(token_stride=63), dict(token_stride=72),
              dict(head_stride=1000), dict(page_stride=2040), dict(page_stride=1 << 62),
              dict(token_stride=-64), dict(scale_token_stride=0), dict(scale_head_stride=15),
              dict(scale_page_stride=31), dict(scale_page_stride=1 << 62)]


@pytest.mark.parametrize("change", BAD_CACHES, ids=str)
def test_bad_caches_are_refused(lib, change):
    for call in (append, attend):
        rc, err = call(lib, cache(**change), batch())
        assert rc != 0 and err.message, change
    assert lib.et_b200_paged_attention8_workspace_bytes_v1(C.byref(cache(**change)), 4) == 0


@pytest.mark.parametrize("change", BAD_BATCHES + [dict(offsets=FAKE + 4), dict(lengths=FAKE + 4),
                                                  dict(page_table=FAKE + 2), dict(status=FAKE + 1),
                                                  dict(table_columns=(2 ** 31 - 4097) // 16 + 1)], ids=str)
def test_bad_batches_are_refused(lib, change):
    for call in (append, attend):
        rc, err = call(lib, cache(), batch(**change))
        assert rc != 0 and err.message, change


@pytest.mark.parametrize("dtype,size", [(0, 4), (1, 2), (2, 2)])
def test_bad_arguments_are_refused(lib, dtype, size):
    c = cache(dtype=dtype)
    half, empty = paged.RopeDescriptor(FAKE, None, 10), paged.RopeDescriptor(FAKE, FAKE, 0)
    off = paged.RopeDescriptor(FAKE + 2, FAKE, 10)
    for kw in (dict(k=None), dict(v=None), dict(ks=127), dict(vs=64), dict(k=FAKE + size // 2),
               dict(v=FAKE + 1), dict(ks=1 << 40), dict(rope=half), dict(rope=empty), dict(rope=off)):
        assert append(lib, c, batch(), **kw)[0] != 0, kw
    for kw in (dict(q=None), dict(o=None), dict(qs=255), dict(os=255), dict(q=FAKE + size // 2),
               dict(o=FAKE + 1), dict(lse=FAKE + 2), dict(heads=0), dict(heads=3), dict(heads=65538),
               dict(ws=None), dict(ws=FAKE + 16), dict(size=64), dict(rope=half), dict(rope=empty),
               dict(rope=off)):
        assert attend(lib, c, batch(), **kw)[0] != 0, kw
    assert append(lib, None, batch())[0] != 0 and append(lib, c, None)[0] != 0
    assert attend(lib, None, batch())[0] != 0 and attend(lib, c, None)[0] != 0


def test_empty_steps_do_nothing(lib):
    for b in (batch(tokens=0), batch(batch=0)):
        assert append(lib, cache(), b, k=None, v=None)[0] == 0
        assert attend(lib, cache(), b, q=None, o=None, ws=None, size=0)[0] == 0


def probabilities(lib, logits=FAKE, probs=FAKE + (1 << 20), stride=100, **change):
    d = dict(struct_size=C.sizeof(sampling.SamplingDescriptor), rows=2, vocabulary=100,
             row_stride=100, dtype=0, reserved=0, temperature=None, top_k=None, top_p=None,
             min_p=None)
    d.update(change)
    s = sampling.SamplingDescriptor(*[d[f] for f, _ in sampling.SamplingDescriptor._fields_])
    err = k1.KernelError()
    return lib.et_b200_probabilities_v1(C.byref(s), logits, probs, stride, None, C.byref(err)), err


def test_bad_distributions_are_refused(lib):
    for kw in (dict(struct_size=8), dict(rows=-1), dict(vocabulary=0), dict(vocabulary=(1 << 22) + 1),
               dict(row_stride=99), dict(dtype=3), dict(logits=None), dict(probs=None), dict(stride=99),
               dict(stride=1 << 40), dict(logits=FAKE + 2), dict(probs=FAKE + 2), dict(top_k=FAKE + 4),
               dict(temperature=FAKE + 2), dict(top_p=FAKE + 1), dict(min_p=FAKE + 3)):
        rc, err = probabilities(lib, **kw)
        assert rc != 0 and err.message, kw
    assert lib.et_b200_probabilities_v1(None, FAKE, FAKE, 100, None, None) != 0
    assert probabilities(lib, rows=0, logits=None, probs=None)[0] == 0


def test_distributions_over_their_logits_are_refused(lib):
    """Zeros go out while logits are read: no byte of a row may belong to both."""
    for kw in (dict(probs=FAKE), dict(probs=FAKE + 4), dict(probs=FAKE + 4 * 199), dict(probs=FAKE - 4 * 99),
               dict(probs=FAKE + 400, row_stride=150, stride=150), dict(probs=FAKE + 400, row_stride=200),
               dict(probs=FAKE, dtype=1), dict(probs=FAKE, rows=1)):
        rc, err = probabilities(lib, **kw)
        assert rc != 0 and b"overlap" in err.message, kw


def verify(lib, target=FAKE, draft=FAKE, ids=FAKE, accepted=FAKE, **change):
    d = dict(struct_size=C.sizeof(sampling.VerificationDescriptor), batch=2, tokens=6, vocabulary=100,
             target_stride=100, draft_stride=100, offsets=FAKE, drafts=FAKE, accept_uniform=FAKE,
             draw_uniform=FAKE, status=None)
    d.update(change)
    s = sampling.VerificationDescriptor(*[d[f] for f, _ in sampling.VerificationDescriptor._fields_])
    err = k1.KernelError()
    return lib.et_b200_verify_v1(C.byref(s), target, draft, ids, accepted, None, C.byref(err)), err


def test_bad_verifications_are_refused(lib):
    for kw in (dict(struct_size=8), dict(batch=-1), dict(batch=(1 << 20) + 1), dict(tokens=-1),
               dict(tokens=(1 << 26) + 1), dict(vocabulary=0), dict(vocabulary=(1 << 22) + 1),
               dict(target_stride=99), dict(target_stride=1 << 40), dict(draft_stride=99),
               dict(target=None), dict(ids=None), dict(accepted=None), dict(offsets=None),
               dict(drafts=None), dict(accept_uniform=None), dict(draw_uniform=None),
               dict(target=FAKE + 2), dict(draft=FAKE + 1), dict(ids=FAKE + 4), dict(accepted=FAKE + 4),
               dict(offsets=FAKE + 4), dict(drafts=FAKE + 4), dict(accept_uniform=FAKE + 2),
               dict(draw_uniform=FAKE + 1), dict(status=FAKE + 2)):
        rc, err = verify(lib, **kw)
        assert rc != 0 and err.message, kw
    assert lib.et_b200_verify_v1(None, FAKE, FAKE, FAKE, FAKE, None, None) != 0
    assert verify(lib, batch=0, tokens=0, target=None, ids=None, accepted=None, offsets=None)[0] == 0


def test_the_plain_quantisation_is_the_types():
    """The plain form that the GPU tests compare with, against torch's own e4m3 type."""
    table = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mine = e4m3_values()
    assert torch.equal(torch.isnan(table), torch.isnan(mine))
    assert torch.equal(table[~torch.isnan(table)], mine[~torch.isnan(mine)])
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2000, 16, generator=g) * torch.exp2(torch.randint(-140, 120, (2000, 1), generator=g).float())
    x[::50] = 0.0
    bits, s = quantise(x)
    want = (x.double() / torch.where(s > 0, s, 1.0).double()[:, None]).float().to(torch.float8_e4m3fn)
    assert torch.equal(bits, want.view(torch.uint8))
    top = x.double().abs().amax(1)
    assert (top <= 448.0 * s.double()).all() and (s[top == 0] == 0).all()
    assert ((448.0 * s.double() / 2 < top) | (s == 2.0 ** -126) | (top == 0)).all()
