"""What the paged operators and sample_tokens refuse of tensors on the GPU: nothing is launched."""
import pytest
import torch

import transformer_amd as T

pytestmark = pytest.mark.gpu


def bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16, device="cuda")


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32, device="cuda")


def good():
    pages, scales = T.new_paged_cache(4, 16, 512, bits=4)
    return dict(q_lat=bf(2, 16, 512), q_rope=bf(2, 16, 64), pages=pages, scales=scales, block_table=i32(2, 2), seq_lens=i32(2), scale=0.1)


DECODE = [
    "q_lat dtype", "q_lat shape", "q_rope shape", "pages dtype", "pages shape", "no scales", "scales shape", "scales dtype", "table dtype", "table rows",
    "lens dtype", "lens shape", "rope heads", "scale", "cpu lens", "rows apart", "misaligned",
]


@pytest.mark.parametrize("what", DECODE)
def test_decode_refusals(what):
    a = good()
    flat = torch.zeros(4 * 16 * 288 + 8, dtype=torch.uint8, device="cuda")
    a.update({
        "q_lat dtype": dict(q_lat=a["q_lat"].float()), "q_lat shape": dict(q_lat=bf(2, 16, 384)), "q_rope shape": dict(q_rope=bf(2, 16, 32)), "pages dtype": dict(pages=bf(4, 16, 288)),
        "pages shape": dict(pages=a["pages"][0]), "no scales": dict(scales=None), "scales shape": dict(scales=bf(4, 16, 9)),
        "scales dtype": dict(scales=a["scales"].float()), "table dtype": dict(block_table=a["block_table"].long()),
        "table rows": dict(block_table=i32(3, 2)), "lens dtype": dict(seq_lens=a["seq_lens"].long()), "lens shape": dict(seq_lens=i32(2, 1)),
        "rope heads": dict(q_lat=bf(2, 16, 384), q_rope=bf(2, 16, 64)), "scale": dict(scale=0.0), "cpu lens": dict(seq_lens=a["seq_lens"].cpu()),
        "rows apart": dict(pages=torch.zeros(4, 16, 304, dtype=torch.uint8, device="cuda")[..., :288]),
        "misaligned": dict(pages=flat[8:].view(4, 16, 288)),
    }[what])
    with pytest.raises((ValueError, TypeError, RuntimeError)):
        T.paged_decode(**a)


def test_append_refusals():
    pages, scales = T.new_paged_cache(4, 16, 512, bits=4)
    ok = dict(qk=bf(2, 3, 17, 64), c_new=bf(2, 3, 512), pages=pages, scales=scales, cos=bf(8, 32), sin=bf(8, 32), block_table=i32(2, 2),
              starts=i32(2), counts=i32(2))
    assert T.paged_append(**ok).shape == (2, 3, 16, 64)
    for change in (dict(qk=bf(2, 3, 0, 64)), dict(qk=bf(2, 3, 17, 32)), dict(qk=bf(2, 2, 17, 64)), dict(c_new=bf(2, 3, 400)), dict(cos=bf(8, 64)),
                   dict(sin=bf(9, 32)), dict(cos=bf(8, 32).float()), dict(starts=i32(3)), dict(starts=i32(2).float()), dict(counts=i32(2).long()),
                   dict(block_table=i32(2)), dict(scales=None), dict(starts=i32(2).cpu())):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            T.paged_append(**{**ok, **change})


def test_read_and_sample_refusals():
    pages, scales = T.new_paged_cache(4, 16, 512, bits=4)
    for args in ((pages, scales, i32(2, 2), 512, -1), (pages, scales, i32(2, 2), 500, 4), (pages, scales, i32(2, 2).float(), 512, 4),
                 (pages, None, i32(2, 2), 512, 4), (pages, scales, i32(2, 2), 512, 4, i32(3))):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            T.paged_read(*args)
    x, u = torch.zeros(2, 9, device="cuda"), torch.zeros(2, device="cuda")
    for args, kw in (((x[0], u), {}), ((x, u[:1]), {}), ((x.half(), u), {}), ((x, u.double()), {}), ((x, u.cpu()), {}), ((x[:, :0], u), {}),
                     ((x, u), dict(top_k=u)), ((x, u), dict(temperature=u[:1])), ((x, u), dict(top_p=u.double())),
                     ((x, u), dict(min_p=u.cpu()))):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            T.sample_tokens(*args, **kw)
