"""Calls of the paged-cache operators whose arguments are unusual.  On the CPU a call that is not refused for them is refused for its device."""
import pytest
import torch

from vits_amd import ops


def i32(*values):
    return torch.tensor(values, dtype=torch.int32)


def test_caches_of_one_page_need_no_common_stride():
    """Strides of dimensions of one element say nothing, so two caches may differ there; elsewhere they may not."""
    both = torch.zeros(3, 2, 2, 16, 64)
    q, k, v = torch.zeros(2, 4, 64), torch.zeros(2, 2, 64), torch.zeros(2, 2, 64)
    freq = ops.rotary_frequencies(64, device="cpu")
    for k_cache, v_cache, word in ((both[:1, 0], torch.zeros(1, 2, 16, 64), "GPU"), (both[:1, 0], both[1:2, 1], "GPU"), (both[:, 0], torch.zeros(3, 2, 16, 64), "alike")):
        with pytest.raises(ValueError, match=word):
            ops.paged_attention(q, k_cache, v_cache, i32(0)[None], i32(0, 0), i32(3, 4))
        with pytest.raises(ValueError, match=word):
            ops.rotary_store(q, k, v, k_cache, v_cache, i32(3, 4), torch.arange(2), freq)
    one = torch.zeros(3, 1, 16, 64)
    other = torch.zeros(3, 1024, dtype=torch.float32).as_strided((3, 1, 16, 64), (1024, 7, 64, 1))
    with pytest.raises(ValueError, match="GPU"):
        ops.paged_attention(q, one, other, i32(0)[None], i32(0, 0), i32(3, 4))


def rotary_arguments():
    q, k, v = torch.zeros(2, 4, 64), torch.zeros(2, 2, 64), torch.zeros(2, 2, 64)
    caches = torch.zeros(2, 3, 2, 16, 64)
    return dict(q=q, k=k, v=v, k_cache=caches[0], v_cache=caches[1], position=i32(3, 4), slot=torch.arange(2), freq=ops.rotary_frequencies(64, device="cpu"))


def test_an_error_of_an_argument_is_that_error():
    class Odd:
        def __bool__(self):
            raise KeyError("odd")
    with pytest.raises(KeyError):
        ops.rotary_store(**rotary_arguments(), interleaved=Odd())
    for bad in ("1.5", None, [1.0]):
        with pytest.raises(TypeError):
            ops.rotary_store(**rotary_arguments(), scale=bad)


def test_what_is_no_tensor_is_a_value_error():
    """The first argument too, whose shape and device the functions look at themselves."""
    r = rotary_arguments()
    pages = ops.new_pages(3, 4, 20, device="cpu")
    for bad in (None, [1.0, 2.0], 3):
        with pytest.raises(ValueError, match="q must be a tensor"):
            ops.paged_attention(bad, r["k_cache"], r["v_cache"], i32(0)[None], i32(0, 0), i32(3, 4))
        with pytest.raises(ValueError, match="lengths must be a tensor"):
            ops.page_plan(bad, i32(1, 1, 1), pages.table, pages.ring, pages.cursor, 16, rows=4)
        if bad is not None:
            with pytest.raises(ValueError, match="q must be a tensor"):
                ops.rotary_store(**{**r, "q": bad})
            with pytest.raises(ValueError, match="k must be a tensor"):
                ops.rotary_store(**{**r, "q": None, "k": bad})
    with pytest.raises(ValueError, match="q must be"):
        ops.paged_attention(torch.zeros(()), r["k_cache"], r["v_cache"], i32(0)[None], i32(0, 0), i32(3, 4))
    with pytest.raises(ValueError, match="out"):
        ops.page_plan(pages.lengths, i32(1, 1, 1), pages.table, pages.ring, pages.cursor, 16, out=[None] * 7)
