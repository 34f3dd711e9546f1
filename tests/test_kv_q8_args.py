"""Refusals of the 8-bit cache, attention and draft-verification entry points
(argument checks come before any GPU work, so they run without one)."""
import ctypes as C

import numpy as np
import pytest

from eosllm_b200 import backend as B


@pytest.fixture()
def buf():
    raw = np.zeros(1 << 16, np.uint8)
    off = (-raw.ctypes.data) % 256
    a = raw[off:off + (1 << 15)]
    assert a.ctypes.data % 256 == 0
    return a


def pool(buf, n_pages=2, kvh=2, hd=128):
    return B.kv_q8_pool(buf, n_pages, kvh, hd)


def copy_status(lib, name, p, k, v, stride, n_rows, row0, table, ts, pos, n_seq):
    return getattr(lib, name)(C.byref(p) if p is not None else None, k, v, stride, n_rows, row0, table, ts, pos, n_seq,
                              None)


@pytest.mark.parametrize("name", ["eosi_cuda_kv_q8_write_dev", "eosi_cuda_kv_q8_read_dev"])
def test_copy_refusals(cuda_lib, buf, name):
    a = buf.ctypes.data
    ok = dict(p=pool(buf), k=a, v=a, stride=256, n_rows=4, row0=a, table=a, ts=1, pos=a, n_seq=2)

    def st(**kw):
        return copy_status(cuda_lib, name, **{**ok, **kw})

    assert st(p=None) == B.EOS_E_INVALID_ARG
    for field in ("k", "v", "table", "pos"):
        assert st(**{field: None}) == B.EOS_E_INVALID_ARG, field
    assert st(k=a + 4) == B.EOS_E_INVALID_ARG
    assert "16-byte" in B.last_error()
    assert st(stride=255) == B.EOS_E_INVALID_ARG      # not a multiple of 4
    assert st(stride=252) == B.EOS_E_INVALID_ARG      # rows of 2 * 128 do not fit
    assert st(row0=None, n_rows=5) == B.EOS_E_INVALID_ARG  # 5 rows of 2 equal sequences
    assert st(p=pool(buf, hd=96)) == B.EOS_E_UNSUPPORTED
    assert st(p=pool(buf, kvh=0)) == B.EOS_E_INVALID_ARG
    assert st(p=B.kv_q8_pool(a + 8, 2, 2, 128)) == B.EOS_E_INVALID_ARG
    assert st(ts=1 << 26) == B.EOS_E_INVALID_ARG
    assert st(n_rows=1 << 31, row0=a) == B.EOS_E_INVALID_ARG
    # nothing to do needs no GPU
    assert st(n_rows=0) == B.EOS_OK and st(n_seq=0) == B.EOS_OK


def test_page_bytes(cuda_lib):
    for kvh, hd in ((1, 64), (8, 128), (3, 256)):
        assert B.kv_q8_page_bytes(kvh, hd) == kvh * (2 * 128 * hd + 128 * 8)


def test_attention_refusals(cuda_lib, buf):
    a = buf.ctypes.data
    base = dict(table=a, table_stride=2, seq_len=a, max_len=256, n_seq=2, n_rows=4, max_rows=2, row0=a, prefix_table=a,
                prefix_len=a, max_prefix=100)

    def st(p=None, n_head=4, q=a, qs=512, out=a, os_=512, scratch=a, nbytes=1 << 40, scale=0.1, **kw):
        p = pool(buf) if p is None else p
        b = B.attn_batch(**{**base, **kw})
        return cuda_lib.eosi_cuda_kv_q8_attn_dev(C.byref(p), C.byref(b), q, qs, out, os_, n_head, scale, scratch, nbytes,
                                                 None)

    assert st(n_head=3) == B.EOS_E_INVALID_ARG         # not a multiple of the 2 kv heads
    assert st(n_head=0) == B.EOS_E_INVALID_ARG
    assert st(scale=float("nan")) == B.EOS_E_INVALID_ARG and st(scale=float("inf")) == B.EOS_E_INVALID_ARG
    assert st(qs=508) == B.EOS_E_INVALID_ARG and st(qs=514) == B.EOS_E_INVALID_ARG and st(os_=508) == B.EOS_E_INVALID_ARG
    for kw in (dict(q=None), dict(out=None), dict(scratch=None), dict(seq_len=None), dict(table=None),
               dict(prefix_table=None), dict(prefix_len=None)):
        assert st(**kw) == B.EOS_E_INVALID_ARG, kw
    assert st(q=a + 4) == B.EOS_E_INVALID_ARG and st(scratch=a + 8) == B.EOS_E_INVALID_ARG
    assert st(max_rows=0) == B.EOS_E_INVALID_ARG and st(max_rows=5) == B.EOS_E_INVALID_ARG
    assert st(row0=None, max_rows=1) == B.EOS_E_INVALID_ARG  # two rows a sequence
    assert st(row0=None, n_rows=3) == B.EOS_E_INVALID_ARG
    assert st(max_len=257) == B.EOS_E_INVALID_ARG      # beyond two pages
    assert st(n_seq=1025) == B.EOS_E_UNSUPPORTED
    assert st(p=pool(buf, hd=32)) == B.EOS_E_UNSUPPORTED
    assert st(nbytes=0) == B.EOS_E_INVALID_ARG and "scratch" in B.last_error()
    assert st(n_rows=0) == B.EOS_OK and st(n_seq=0, n_rows=0) == B.EOS_OK
    # the scratch size: 0 for arguments that would be refused
    b = B.attn_batch(**base)
    assert B.kv_q8_attn_scratch_bytes(pool(buf), b, 4) > 0
    assert B.kv_q8_attn_scratch_bytes(pool(buf), b, 3) == 0


def test_verify_refusals(cuda_lib, buf):
    a = buf.ctypes.data

    def st(p=a, q=a, stride=100, drafts=a, n_draft=None, kk=2, u=a, n_seq=1, vocab=100, tokens=a, n_tokens=a):
        return cuda_lib.eosi_cuda_verify_draft_dev(p, q, stride, drafts, n_draft, kk, u, n_seq, vocab, tokens,
                                                   n_tokens, None)

    for kw in (dict(p=None), dict(q=None), dict(drafts=None), dict(u=None), dict(tokens=None), dict(n_tokens=None),
               dict(stride=99), dict(vocab=0), dict(kk=1 << 20), dict(vocab=1 << 31, stride=1 << 31)):
        assert st(**kw) == B.EOS_E_INVALID_ARG, kw
    assert st(n_seq=0) == B.EOS_OK


def test_decoder_refusals_without_a_decoder(cuda_lib):
    for name, args in (("eosi_cuda_text_set_cache", (None, 1)), ("eosi_cuda_text_fork", (None, 2, 4, 0)),
                       ("eosi_cuda_text_branch_step", (None, None, 0, None, None, 1.0, None, None)),
                       ("eosi_cuda_text_branch_adopt", (None, 0)), ("eosi_cuda_text_branch_close", (None,))):
        assert getattr(cuda_lib, name)(*args) == B.EOS_E_INVALID_ARG, name
    assert cuda_lib.eosi_cuda_text_cache(None) == 0
