"""What of the paged 4-bit cache needs no GPU: the plain model's layout, page sizes, null arguments."""
import numpy as np
import pytest

import b200attn
import kv4_helpers as kv


@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_layout_places_every_code_once_and_round_trips(D):
    kb, vb, shift, param = kv.places(D)
    for byte in (kb, vb):
        assert len({(int(a), int(s)) for a, s in zip(byte.ravel(), shift.ravel())}) == 16 * D
        assert byte.min() == 0 and byte.max() == 8 * D - 1
        # a byte holds codes of one key: rows are stored independently
        owner = {}
        for key in range(16):
            for a in byte[key]:
                assert owner.setdefault(int(a), key) == key
    assert sorted(param.ravel()) == list(range(16 * D // 32))
    rng = np.random.default_rng(D)
    x = rng.standard_normal((2, 3, 32, D)).astype(np.float32)
    c, s = kv.quantise(x)
    raw = kv.pack(c, s, c[::-1], s[::-1])
    assert raw.shape == (2, 3, 40 * D)
    for a, b in zip(kv.unpack(raw, D), (c, s, c[::-1], s[::-1])):
        np.testing.assert_array_equal(a, b)
    # half a step (with s rounded to fp16: 15 * 2^-11 of one more) and z's rounding
    g = x.reshape(2, 3, 32, -1, 32)
    step = s[..., 0].astype(np.float64)[..., None]
    err = np.abs(kv.values(c, s).reshape(g.shape) - g)
    assert np.all(err <= step * (0.5 + 16 * 2.0 ** -11) + np.abs(g.min(-1, keepdims=True)) * 2.0 ** -10)


def test_page_bytes():
    assert b200attn.kv4_page_bytes(2, 64, 32) == 2 * 32 * 64 * 5 // 4
    assert b200attn.kv4_page_bytes(1, 256, 16) == 16 * 320
    for bad in ((0, 64, 32), (2, 80, 32), (2, 64, 24), (2, 64, 0), (2, 64, 2048)):
        with pytest.raises(ValueError):
            b200attn.kv4_page_bytes(*bad)


def test_calls_with_null_context_are_rejected():
    lib = b200attn.lib()
    assert lib.b2a_kv4_append(None, None, 1, None, None, 0, None, None, 1, 1, 0, 0.0, None, 0.0, None, None, None) == \
        b200attn.B2A_EINVAL
    assert lib.b2a_kv4_attention(None, None, 1, None, 0, None, None, 1, 1, 1, 0.1, 0, 0.0, 0, None, 0.0, None, None) == \
        b200attn.B2A_EINVAL
    assert lib.b2a_kv4_decode(None, None, 1, None, 0, None, None, 0, None, None, 1, 1, 1, 0.1, 0, 0.0, 0, None, None,
                              0.0, None, None, None, None) == b200attn.B2A_EINVAL
    assert lib.b2a_pages_fork(None, None, None, None) == b200attn.B2A_EINVAL
    assert lib.b2a_pages_free(None, None, None, None, 16, None) == b200attn.B2A_EINVAL
    assert lib.b2a_pages_reserve(None, None, None, None, 16, None, None) == b200attn.B2A_EINVAL
    assert lib.b2a_pages_compact(None, None, None, None) == b200attn.B2A_EINVAL
