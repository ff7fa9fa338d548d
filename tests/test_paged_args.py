"""The paged cache's and the sampling's entry points refuse bad arguments on the host: no pointer is followed, nothing is launched, so
these run without a GPU.  So do the checks of the public functions, on tensors without storage."""
import ctypes
import math

import pytest
import torch

import transformer_amd as T
from transformer_amd import _lib

CACHE = dict(pages=4096, scales=8192, block_table=12288, n_pages=10, page_size=16, page_stride=16 * 288, scale_stride=16 * 9,
             table_pages=4, table_stride=4, d_latent=512, n_k_rope_heads=1)
ST = _lib.Strides(17 * 64, 17 * 64, 64)
BASE = {
    "mla_paged_append": (_lib.PagedAppendArgs, dict(qk=4096, c_new=4096, q_out=4096, cos=4096, sin=4096, starts=4096, counts=None, B=2,
                                                    T=1, H=16, table_rows=100, qk_stride=ST, c_new_sb=512, c_new_st=512)),
    "mla_paged_read": (_lib.PagedReadArgs, dict(latent=4096, k_rope=4096, starts=None, counts=None, B=2, T=5)),
    "mla_paged_decode": (_lib.PagedDecodeArgs, dict(q_lat=4096, q_rope=4096, seq_lens=4096, ctx=4096, lse=4096, workspace=4096,
                                                    workspace_bytes=1 << 30, B=2, H=16, q_lat_sb=8192, q_lat_sh=512, q_rope_sb=1024,
                                                    q_rope_sh=64, scale=0.1)),
}
BAD_CACHE = (dict(pages=None), dict(pages=4104), dict(scales=8196), dict(block_table=None), dict(block_table=2), dict(n_pages=-1),
             dict(n_pages=1 << 31), dict(page_size=0), dict(page_size=24), dict(page_size=8192), dict(page_stride=16 * 272),
             dict(page_stride=16 * 288 + 8), dict(scale_stride=100), dict(scale_stride=16 * 9 + 4), dict(table_pages=-1),
             dict(table_pages=1 << 27), dict(table_stride=-4), dict(d_latent=192), dict(d_latent=0), dict(n_k_rope_heads=0),
             dict(n_k_rope_heads=2000))
BAD = {
    "mla_paged_append": (dict(B=-1), dict(T=-1), dict(H=-1), dict(T=1 << 24), dict(B=1 << 24), dict(qk=None), dict(c_new=None), dict(cos=8),
                         dict(sin=None), dict(q_out=None), dict(q_out=4100), dict(starts=None), dict(starts=4098), dict(counts=4097),
                         dict(c_new_sb=-8), dict(c_new_st=12), dict(qk_stride=_lib.Strides(4, 64, 64)), dict(table_rows=-1),
                         dict(B=(1 << 24) - 1, T=(1 << 24) - 1)),
    "mla_paged_read": (dict(B=-1), dict(T=-2), dict(latent=None), dict(k_rope=None), dict(latent=4104), dict(starts=3), dict(counts=2),
                       dict(B=(1 << 24) - 1, T=(1 << 24) - 1)),
    "mla_paged_decode": (dict(workspace_bytes=1000), dict(workspace=4100), dict(B=-1), dict(H=0), dict(H=2000), dict(B=1 << 20), dict(q_lat=None), dict(q_rope=4100), dict(ctx=None), dict(ctx=4104),
                         dict(lse=None), dict(lse=4098), dict(seq_lens=None), dict(seq_lens=4099), dict(q_lat_sb=-8), dict(q_rope_sh=12),
                         dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf)),
}


@pytest.mark.parametrize("entry", sorted(BASE))
def test_bad_arguments_are_refused(entry):
    lib = _lib.load()
    struct, good = BASE[entry]
    for cache, change in [(c, {}) for c in BAD_CACHE] + [({}, c) for c in BAD[entry]]:
        a = struct(cache=_lib.PagedCache(**{**CACHE, **cache}), **{**good, **change})
        rc = getattr(lib, entry)(ctypes.byref(a), None)
        assert rc < 0 and entry.encode() in lib.mla_last_error(), (entry, cache, change, rc)
    assert getattr(lib, entry)(None, None) == _lib.MLA_ERR_INVALID_ARG
    # without sequences there is nothing to do
    a = struct(cache=_lib.PagedCache(**CACHE), **{**good, "B": 0})
    assert getattr(lib, entry)(ctypes.byref(a), None) == _lib.MLA_OK


def test_rope_heads_go_with_the_query_heads():
    lib = _lib.load()
    struct, good = BASE["mla_paged_decode"]
    a = struct(cache=_lib.PagedCache(**{**CACHE, "n_k_rope_heads": 3, "page_stride": 1 << 20, "scale_stride": 1 << 20}), **good)
    assert lib.mla_paged_decode(ctypes.byref(a), None) == _lib.MLA_ERR_INVALID_ARG


SAMPLE = dict(logits=4096, u=4096, temperature_rows=None, top_k_rows=None, top_p_rows=None, min_p_rows=None, tokens=4096, logprobs=4096,
              B=2, V=100, stride=100, temperature=1.0, top_p=1.0, min_p=0.0, top_k=0, dtype=0)


def test_bad_sampling_arguments_are_refused():
    lib = _lib.load()
    for change in (dict(B=-1), dict(V=0), dict(V=(1 << 19) + 1), dict(logits=None), dict(u=None), dict(tokens=None), dict(logprobs=None),
                   dict(logits=4097), dict(dtype=1, logits=4098), dict(tokens=4100), dict(u=4098), dict(logprobs=4097), dict(stride=-1),
                   dict(dtype=2), dict(temperature=math.nan), dict(top_p=math.nan), dict(min_p=math.nan), dict(temperature_rows=4098),
                   dict(top_k_rows=4097), dict(top_p_rows=2), dict(min_p_rows=3)):
        a = _lib.SampleArgs(**{**SAMPLE, **change})
        assert lib.mla_sample(ctypes.byref(a), None) < 0 and b"mla_sample" in lib.mla_last_error(), change
    assert lib.mla_sample(None, None) == _lib.MLA_ERR_INVALID_ARG
    assert lib.mla_sample(ctypes.byref(_lib.SampleArgs(**{**SAMPLE, "B": 0})), None) == _lib.MLA_OK


def bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def test_public_functions_refuse_the_cpu():
    pages, scales = T.new_paged_cache(2, 16, 512, bits=4, device="cpu")
    table, n = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: T.paged_decode(bf(1, 16, 512), bf(1, 16, 64), pages, scales, table, n, 0.1),
                 lambda: T.paged_append(bf(1, 1, 17, 64), bf(1, 1, 512), pages, scales, bf(8, 32), bf(8, 32), table, n),
                 lambda: T.paged_read(pages, scales, table, 512, 4),
                 lambda: T.sample_tokens(torch.zeros(2, 8), torch.zeros(2))):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_new_cache_layouts():
    pages, scales = T.new_paged_cache(3, 32, 384, 14, 16, device="cpu")
    assert pages.shape == (3, 32, 1280) and pages.dtype == torch.bfloat16 and scales is None
    pages, scales = T.new_paged_cache(3, 32, 384, 14, 4, device="cpu")
    assert pages.shape == (3, 32, 640) and pages.dtype == torch.uint8 and scales.shape == (3, 20, 32) and scales.dtype == torch.bfloat16
    for kw in (dict(bits=8), dict(size=24), dict(size=0), dict(d_latent=100), dict(n_k_rope_heads=0), dict(n_pages=-1)):
        with pytest.raises(ValueError):
            T.new_paged_cache(**{**dict(n_pages=1, size=16, d_latent=512, device="cpu"), **kw})


def test_settings_are_checked():
    x, u = torch.zeros(2, 8), torch.zeros(2)
    for kw in (dict(temperature=math.nan), dict(top_k=1.5), dict(top_k=1 << 40), dict(top_p=math.nan), dict(min_p=True)):
        with pytest.raises(ValueError, match="sample_tokens"):
            T.sample_tokens(x, u, **kw)
