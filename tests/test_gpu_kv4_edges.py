"""Edges of the paged 4-bit KV cache that the model's cases do not reach."""
import numpy as np
import pytest

import oracle
from helpers import to_np
from test_gpu_kv4 import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", [oracle.F16, oracle.BF16])
def test_prompt_store_clamps_a_tie_at_the_top(ctx, D, dtype):
    """Groups of multiples of 2^-24 from 0 to 31: s rounds to 2 * 2^-24, so the largest element scales to 15.5,
    which rounds to 16 and is held as 15.  All of it is exact, the held rows too (c * 2^-23)."""
    import b200attn
    c = Case(ctx=[0, 7], T=20, Hq=2, Hkv=2, D=D, page=48, dtype=dtype, rope=None, seed=D)
    rng = np.random.default_rng(D)
    for name in ("k", "v"):
        x = rng.integers(0, 32, c.k.shape)
        x[..., 0::32], x[..., 21::32] = 0, 31
        setattr(c, name, (x * 2.0 ** -24).astype(np.float32))
    t = c.device()
    b200attn.kv4_append(ctx, t["k"], t["v"], t["pages"], t["table"], t["ctx"], k_held=t["k_held"], v_held=t["v_held"],
                        **c.more())
    ctx.check_device_status()
    _, _, kh, vh = c.expect()
    c.check_pages(t["pages"].cpu().numpy(), exact=True)
    np.testing.assert_array_equal(to_np(t["k_held"]), kh)
    np.testing.assert_array_equal(to_np(t["v_held"]), vh)


@pytest.mark.parametrize("page,slots,L", [(48, 3, 100), (16, 10, 97), (16, 9, 144)])
def test_lengths_past_the_table_but_inside_its_last_tile(ctx, page, slots, L):
    """A chunk's rows are staged for whole tiles of 128 keys; lengths between the table's room and the tile's end
    do not fit all the same: NaN, nothing stored, the other sequences as ever."""
    import torch
    import b200attn
    c = Case(ctx=[20, 60, 50], T=70, Hq=4, Hkv=2, D=64, page=page, dtype=oracle.BF16, seed=page)
    c.table = np.pad(c.table, ((0, 0), (0, max(0, slots - c.table.shape[1]))), constant_values=-1)[:, :slots]
    room = slots * page
    assert room < L + c.T <= -(-room // 128) * 128
    t = c.device()
    b200attn.kv4_decode(ctx, t["q"], t["k"], t["v"], t["pages"], t["table"], t["ctx"], t["o"], c.scale, **c.more())
    ctx.check_device_status()
    o, tol, _, _ = c.expect()
    c.check_out(to_np(t["o"]), o, tol)
    t["ctx"][1] = L
    before = t["pages"].clone()

    def check():
        with pytest.raises(b200attn.B200RuntimeException, match="ctx_lens"):
            ctx.check_device_status()
        assert bool(torch.isnan(t["o"][1]).all())
        c.check_out(to_np(t["o"])[[0, 2]], o[[0, 2]], tol[[0, 2]])
        assert torch.equal(t["pages"], before)

    b200attn.kv4_decode(ctx, t["q"], t["k"], t["v"], t["pages"], t["table"], t["ctx"], t["o"], c.scale, **c.more())
    check()
    t["o"].zero_()
    b200attn.kv4_attention(ctx, t["q"], t["pages"], t["table"], t["ctx"], t["o"], c.scale, **c.more())
    check()
