"""Largest sizes of the serving operators' entry points, on the host."""
import ctypes

import pytest

from transformer_amd import _lib
from tests.test_paged_args import BASE, CACHE, SAMPLE


def decode_args(**change):
    cache = {k: change.pop(k) for k in list(change) if k in CACHE}
    struct, good = BASE["mla_paged_decode"]
    return struct(cache=_lib.PagedCache(**{**CACHE, **cache}), **{**good, **change})


@pytest.mark.parametrize("d_latent", [64, 512])
@pytest.mark.parametrize("scales", [None, 8192])
@pytest.mark.parametrize("B,H", [(1, 1), (64, 16), ((1 << 20) - 1, 16), ((1 << 20) - 1, 1024), (300, 33)])
def test_the_workspace_goes_by_sizes(B, H, scales, d_latent):
    """At most 17 MB and 4 bytes a unit (a sequence and 16 heads), for every size that is taken."""
    a = decode_args(B=B, H=H, scales=scales, d_latent=d_latent, table_pages=1, page_stride=1 << 20, scale_stride=1 << 20)
    n = _lib.load().mla_paged_decode_workspace_bytes(ctypes.byref(a))
    units = 4 * B * ((H + 15) // 16)
    assert units < n <= 17_000_000 + units


@pytest.mark.parametrize("B", [1 << 22, (1 << 31) - 1])
def test_more_rows_than_a_launch_holds_are_refused(B):
    """A row is a workgroup of 1024 threads, and a launch has less than 2^32."""
    lib = _lib.load()
    a = _lib.SampleArgs(**{**SAMPLE, "B": B})
    assert lib.mla_sample(ctypes.byref(a), None) == _lib.MLA_ERR_INVALID_ARG and b"out of range" in lib.mla_last_error()
