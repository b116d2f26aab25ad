"""How the binding reads the rows of a paged 4-bit cache's calls: address and token distance of [B,T,H,D] tensors."""
import pytest
import torch

from b200attn import _token_rows


class Rows:
    """A host tensor that passes for a device one: the binding reads only its shape, strides and address."""

    is_cuda = True

    def __init__(self, t):
        self.t, self.shape = t, t.shape

    def __getattr__(self, name):
        return getattr(self.t, name)


@pytest.mark.parametrize("expand", [
    lambda: torch.zeros(1, 1, 2, 64).expand(3, 1, 2, 64),      # one row for every sequence
    lambda: torch.zeros(1, 1, 2, 64).expand(3, 5, 2, 64),      # for every token too
    lambda: torch.zeros(1, 1, 2, 64).expand(1, 5, 2, 64),
    lambda: torch.zeros(1, 1, 1, 64).expand(4, 1, 1, 64),
    lambda: torch.zeros(512).as_strided((3, 1, 2, 64), (64, 64, 64, 1)),   # overlapping
    lambda: torch.zeros(512).as_strided((1, 3, 2, 64), (64, 64, 64, 1)),
])
def test_rows_that_share_memory_are_refused(expand):
    """The library takes a distance of 0 as dense rows, which would lie past the tensor's memory."""
    t = expand()
    with pytest.raises(ValueError, match="k_new must hold its tokens at least"):
        _token_rows(Rows(t), "k_new", t.shape)


@pytest.mark.parametrize("make,step", [
    (lambda: torch.zeros(3, 5, 2, 64), 128),
    (lambda: torch.zeros(3, 5, 8, 64)[:, :, 2:4], 512),        # a slice of fused rows
    (lambda: torch.zeros(3, 5, 8, 64)[:, 2:3, 2:4], 2560),     # one token of longer rows
    (lambda: torch.zeros(1, 5, 8, 64)[:, :, :2], 512),
    (lambda: torch.zeros(1, 1, 8, 64)[:, :, :2], 128),
    (lambda: torch.zeros(1, 1, 2, 64).expand(1, 1, 2, 64), 128),
])
def test_distances_of_rows_that_are_taken(make, step):
    t = make()
    assert _token_rows(Rows(t), "q", t.shape) == (t.data_ptr(), step)


def test_heads_apart_and_uneven_tokens_are_refused():
    for t in (torch.zeros(3, 5, 8, 64)[:, :, ::2], torch.zeros(3, 6, 2, 64)[:, :5], torch.zeros(3, 5, 2, 128)[..., ::2]):
        with pytest.raises(ValueError, match="one distance"):
            _token_rows(Rows(t), "q", t.shape)


def test_empty_pools_and_rows_are_refused_by_name():
    """Sizes of zero end in the message of the check, not in a division by them."""
    from b200attn import _kv4_cache, _kv4_call_rows, _page_pool
    i32 = lambda *s: Rows(torch.zeros(*s, dtype=torch.int32))
    u8 = lambda *s: Rows(torch.zeros(*s, dtype=torch.uint8))
    for pages in (u8(0, 4, 16), u8(2, 0, 16)):
        with pytest.raises(ValueError, match="at least one layer and one page"):
            _page_pool(i32(3, 5), i32(pages.shape[1]), pages)
    with pytest.raises(ValueError, match="no whole rows"):
        _kv4_cache(u8(4, 2, 640), i32(3, 5), 3, 0, 2)
    rows = Rows(torch.zeros(3, 1, 2, 0, dtype=torch.float16))
    assert _kv4_call_rows(rows, rows, u8(4, 2, 640), i32(3, 5), i32(3), None, None, None, torch.float16, rows.shape) is None
