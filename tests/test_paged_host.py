"""The serving operators' host side on tensors without a GPU: what is taken as it is and what is copied."""
import pytest
import torch

from transformer_amd import _lib, paged
from transformer_amd.host_calls import Entry


def layouts():
    """(name, tensor): dimensions of size 1 whose strides are no multiple of 8, as products and permutes of few rows leave them."""
    flat = torch.arange(1 << 16).to(torch.bfloat16)
    yield "q_lat of one sequence", (torch.ones(16, 512, 64) @ torch.arange(64.0).expand(16, 64)[..., None]).bfloat16().permute(2, 0, 1)
    yield "B = 1", flat.as_strided((1, 16, 512), (1, 512, 1))
    yield "one head", flat.as_strided((4, 1, 64), (64, 3, 1))
    yield "both", flat.as_strided((1, 1, 64), (5, 3, 1))
    yield "qk, T = 1", flat.as_strided((2, 1, 17, 64), (17 * 64, 1, 64, 1))
    yield "qk, one head", flat.as_strided((2, 3, 1, 64), (192, 64, 7, 1))
    yield "c_new of one token", flat.as_strided((1, 1, 512), (1, 1, 1))
    yield "rows off the alignment, B = 1", flat.as_strided((1, 16, 64), (3, 64, 1), 4)
    yield "rows apart by 12", flat.as_strided((1, 16, 8), (1, 12, 1))
    yield "inner stride 2", flat.as_strided((1, 16, 64), (1, 128, 2))
    yield "shared rows", flat.as_strided((4, 16, 64), (0, 64, 1))


@pytest.mark.parametrize("name,t", list(layouts()), ids=[n for n, _ in layouts()])
def test_strides_that_the_entry_points_take(name, t):
    got, strides = paged._strided(t)
    assert torch.equal(got, t)
    assert got.data_ptr() % 16 == 0 and strides[-1] == 1
    assert all(s >= 0 and s % 8 == 0 for s in strides[:-1]), strides
    # and they lead to the same values
    assert torch.equal(torch.as_strided(got, t.shape, strides), t)


def test_what_fits_is_not_copied():
    flat = torch.zeros(1 << 16, dtype=torch.bfloat16)
    for shape, strides in (((1, 16, 512), (1, 512, 1)), ((2, 1, 17, 64), (2000, 3, 64, 1)), ((4, 16, 64), (0, 64, 1))):
        t = flat.as_strided(shape, strides)
        assert paged._strided(t)[0].data_ptr() == t.data_ptr()


def test_an_entry_point_is_called_only_once_it_is_bound_whole(monkeypatch):
    """Another thread's call looks at ``fn`` alone: it must not see a function whose argument types are not set yet (a stream's handle
    would go out as a C int)."""
    entry = Entry("mla_sample", "8P3q3f2i4x", "SampleArgs")
    seen = []

    class Function:
        def __setattr__(self, name, value):
            seen.append((name, entry.fn))
            super().__setattr__(name, value)

    monkeypatch.setattr(_lib, "entry", lambda name: None)
    monkeypatch.setattr(_lib, "load", lambda: {"mla_sample": Function()})
    entry._bind()
    assert {name for name, _ in seen} == {"restype", "argtypes"}
    assert all(fn is None for _, fn in seen) and isinstance(entry.fn, Function)
