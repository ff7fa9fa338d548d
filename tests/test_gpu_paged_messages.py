"""The paged operators' and sample_tokens' refusals say what is wrong: the type of each error and its words."""
import pytest
import torch

import transformer_amd as T
from transformer_amd import _lib
from tests.test_gpu_paged_checks import bf, good, i32

pytestmark = pytest.mark.gpu


def decode_changes(a):
    flat = torch.zeros(4 * 16 * 288 + 8, dtype=torch.uint8, device="cuda")
    return {
        "q_lat dtype": (dict(q_lat=a["q_lat"].float()), TypeError, "q_lat must be bfloat16"),
        "q_rope dtype": (dict(q_rope=a["q_rope"].half()), TypeError, "q_rope must be bfloat16"),
        "q_lat rank": (dict(q_lat=a["q_lat"][None]), ValueError, r"expected q_lat \[B, H, d_latent\]"),
        "q_rope shape": (dict(q_rope=bf(2, 16, 32)), ValueError, r"expected q_lat \[B, H, d_latent\]"),
        "latent": (dict(q_lat=bf(2, 16, 320)), ValueError, "not a latent of 320"),
        "rope heads": (dict(q_lat=bf(2, 16, 384)), ValueError, "3 rotated keys do not go with 16 heads"),
        "pages dtype": (dict(pages=bf(4, 16, 288)), TypeError, "pages must be uint8"),
        "pages rank": (dict(pages=a["pages"][0]), TypeError, "pages must be uint8"),
        "no scales": (dict(scales=None), TypeError, "pages must be bfloat16"),
        "page size": (dict(pages=a["pages"][:, :9].contiguous(), scales=bf(4, 9, 9)), ValueError, "pages of 9 tokens"),
        "scales shape": (dict(scales=bf(4, 16, 9)), ValueError, "scales must be bfloat16"),
        "scales dtype": (dict(scales=a["scales"].float()), ValueError, "scales must be bfloat16"),
        "table dtype": (dict(block_table=a["block_table"].long()), ValueError, "block_table must be int32"),
        "table rows": (dict(block_table=i32(3, 2)), ValueError, "block_table must be int32"),
        "lens dtype": (dict(seq_lens=a["seq_lens"].long()), ValueError, "seq_lens must be int32"),
        "lens shape": (dict(seq_lens=i32(2, 1)), ValueError, "seq_lens must be int32"),
        "rows apart": (dict(pages=torch.zeros(4, 16, 304, dtype=torch.uint8, device="cuda")[..., :288]), ValueError, "must lie close together"),
        "misaligned": (dict(pages=flat[8:].view(4, 16, 288)), ValueError, "16-byte aligned"),
        "cpu lens": (dict(seq_lens=a["seq_lens"].cpu()), RuntimeError, "must be on a ROCm GPU"),
        "no scale": (dict(scale=0.0), _lib.MLAKernelError, "scale"),
        "infinite scale": (dict(scale=float("inf")), _lib.MLAKernelError, "scale"),
        "one page for all": (dict(pages=a["pages"][:1].expand(4, 16, 288)), _lib.MLAKernelError, "page_stride"),
    }


@pytest.mark.parametrize("what", [
    "q_lat dtype", "q_rope dtype", "q_lat rank", "q_rope shape", "latent", "rope heads", "pages dtype", "pages rank", "no scales", "page size",
    "scales shape", "scales dtype", "table dtype", "table rows", "lens dtype", "lens shape", "rows apart", "misaligned", "cpu lens", "no scale",
    "infinite scale", "one page for all"])
def test_decode(what):
    a = good()
    change, error, words = decode_changes(a)[what]
    with pytest.raises(error, match=words):
        T.paged_decode(**{**a, **change})


def test_append():
    pages, scales = T.new_paged_cache(4, 16, 512, bits=4)
    ok = dict(qk=bf(2, 3, 17, 64), c_new=bf(2, 3, 512), pages=pages, scales=scales, cos=bf(8, 32), sin=bf(8, 32), block_table=i32(2, 2),
              starts=i32(2), counts=i32(2))
    for change, error, words in (
            (dict(qk=bf(2, 3, 0, 64)), ValueError, "qk has 0 heads"), (dict(qk=bf(2, 3, 17, 32)), ValueError, "expected qk"),
            (dict(qk=bf(2, 2, 17, 64)), ValueError, "expected qk"), (dict(qk=bf(3, 17, 64)), ValueError, "expected qk"),
            (dict(c_new=bf(2, 3, 400)), ValueError, "not a latent of 400"), (dict(c_new=bf(2, 3, 512).float()), TypeError, "c_new must be bfloat16"),
            (dict(cos=bf(8, 64)), ValueError, "cos and sin must be"), (dict(sin=bf(9, 32)), ValueError, "cos and sin must be"),
            (dict(cos=bf(8, 32).float()), TypeError, "cos must be bfloat16"), (dict(starts=i32(3)), ValueError, "starts must be int32"),
            (dict(starts=i32(2).float()), ValueError, "starts must be int32"), (dict(counts=i32(2).long()), ValueError, "counts must be int32"),
            (dict(block_table=i32(2)), ValueError, "block_table must be int32"), (dict(scales=None), TypeError, "pages must be bfloat16"),
            (dict(starts=i32(2).cpu()), RuntimeError, "must be on a ROCm GPU")):
        with pytest.raises(error, match=words):
            T.paged_append(**{**ok, **change})
    assert not scales.any() and (pages == 0x88).all()


def test_read():
    pages, scales = T.new_paged_cache(4, 16, 512, bits=4)
    for args, error, words in (((pages, scales, i32(2, 2), 512, -1), ValueError, "T must not be negative"),
                               ((pages, scales, i32(2, 2), 500, 4), ValueError, "not a latent of 500"),
                               ((pages, scales, i32(2, 2).float(), 512, 4), ValueError, "block_table must be int32"),
                               ((pages, None, i32(2, 2), 512, 4), TypeError, "pages must be bfloat16"),
                               ((pages, scales, i32(2, 2), 512, 4, i32(3)), ValueError, "starts must be int32"),
                               ((pages, scales, i32(2, 2), 512, 4, None, i32(2).long()), ValueError, "counts must be int32")):
        with pytest.raises(error, match=words):
            T.paged_read(*args)


def test_sampling():
    x, u = torch.zeros(2, 9, device="cuda"), torch.zeros(2, device="cuda")
    for args, kw, error, words in (
            ((x[0], u), {}, ValueError, r"expected logits \[B, V\]"), ((x, u[:1]), {}, ValueError, r"expected logits \[B, V\]"),
            ((x[:, :0], u), {}, ValueError, r"expected logits \[B, V\]"),
            ((torch.zeros(1, (1 << 19) + 1, device="cuda"), u[:1]), {}, ValueError, "V up to 524288"),
            ((x.half(), u), {}, TypeError, "logits must be bfloat16 or float32"), ((x, u.double()), {}, TypeError, "u float32"),
            ((x, u.cpu()), {}, RuntimeError, "must be on a ROCm GPU"), ((x, u), dict(top_k=u), ValueError, "top_k of rows must be int32"),
            ((x, u), dict(temperature=u[:1]), ValueError, "temperature of rows must be float32"),
            ((x, u), dict(top_p=u.double()), ValueError, "top_p of rows must be float32"),
            ((x, u), dict(min_p=u.cpu()), RuntimeError, "must be on a ROCm GPU"), ((x, u), dict(top_k=2.0), ValueError, "top_k must be a whole number"),
            ((x, u), dict(temperature=float("nan")), ValueError, "temperature must be a number")):
        with pytest.raises(error, match=words):
            T.sample_tokens(*args, **kw)
    many = torch.zeros(1, 1, device="cuda").expand(1 << 22, 1)
    with pytest.raises(_lib.MLAKernelError, match="out of range"):
        T.sample_tokens(many, torch.zeros(1 << 22, device="cuda"))
