"""Edges of the paged 4-bit KV cache that the model's cases do not reach."""
import numpy as np
import pytest

import kv4_helpers as kv
import oracle
from helpers import normal, to_np
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


def _hold_nan(c, b, pos, which, head=0, group=1):
    """Position pos of sequence b holds NaN in one key ("k") or value group."""
    page, at = c.table[b, pos // c.page], pos % c.page
    parts = kv.unpack(c.pages[page], c.D)
    parts[1 if which == "k" else 3][head, at, group] = np.nan
    c.pages[page] = kv.pack(*parts)


def _capture(run):
    """A CUDA graph of run(), which has been called before with these sizes."""
    import torch
    torch.cuda.synchronize()
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    return g


def test_replayed_chunks_mark_the_rows_that_see_nan(ctx):
    """Two chunk calls in one graph (two layers).  A value group held as NaN in the second one's cache, then in the
    first one's, then in none: each replay marks what this replay reads."""
    import torch
    import b200attn
    layers = [Case(ctx=[40, 90], T=64, Hq=4, Hkv=2, D=128, dtype=oracle.BF16, rope=None, seed=s) for s in (31, 37)]
    dev = [c.device() for c in layers]

    def run():
        for c, t in zip(layers, dev):
            b200attn.kv4_decode(ctx, t["q"], t["k"], t["v"], t["pages"], t["table"], t["ctx"], t["o"], c.scale, **c.more())

    run()
    clean = [t["pages"].clone() for t in dev]
    g = _capture(run)
    want = [t["o"].clone() for t in dev]
    for bad in (1, 0, None, 0, 1, None):
        for i, (c, t) in enumerate(zip(layers, dev)):
            t["o"].zero_()
            t["pages"].copy_(clean[i])
            if i == bad:
                raw = c.pages.copy()
                _hold_nan(c, 0, 17, "v")
                page = int(c.table[0, 17 // c.page])
                t["pages"][page] = torch.from_numpy(c.pages[page]).cuda()
                c.pages = raw
        g.replay()
        torch.cuda.synchronize()
        for i, t in enumerate(dev):
            nan = torch.zeros_like(t["o"], dtype=torch.bool)
            if i == bad:
                nan[0, :, :2, 32:64] = True  # kv head 0's queries, group 1
            assert torch.equal(torch.isnan(t["o"]), nan), (bad, i)
            assert torch.equal(t["o"][~nan], want[i][~nan]), (bad, i)
    del g
    ctx.check_device_status()


def test_chunks_whose_staged_rows_come_in_slices(ctx):
    """A table so wide that one sequence's staged rows fill a slice: three slices, NaN in the second alone."""
    import torch
    import b200attn
    c = Case(ctx=[40, 90, 7], T=66, Hq=4, Hkv=2, D=64, page=64, dtype=oracle.BF16, rope=None, seed=29,
             extra_slots=40000)
    t = c.device()
    more = dict(c.more(), new_lens=t["new"])
    b200attn.kv4_decode(ctx, t["q"], t["k"], t["v"], t["pages"], t["table"], t["ctx"], t["o"], c.scale, **more)
    ctx.check_device_status()
    o, tol, _, _ = c.expect()
    c.check_out(to_np(t["o"]), o, tol)
    clean = t["o"].clone()
    _hold_nan(c, 1, 50, "v")
    page = int(c.table[1, 50 // c.page])
    t["pages"][page] = torch.from_numpy(c.pages[page]).cuda()
    nan = torch.zeros_like(clean, dtype=torch.bool)
    nan[1, :, :2, 32:64] = True  # kv head 0's queries, group 1
    for run in (lambda: b200attn.kv4_attention(ctx, t["q"], t["pages"], t["table"], t["ctx"], t["o"], c.scale, **more),
                lambda: b200attn.kv4_decode(ctx, t["q"], t["k"], t["v"], t["pages"], t["table"], t["ctx"], t["o"],
                                            c.scale, **more)):
        t["o"].zero_()
        run()
        ctx.check_device_status()
        assert torch.equal(torch.isnan(t["o"]), nan)
        assert torch.equal(t["o"][~nan], clean[~nan])


@pytest.mark.parametrize("D,window", [(64, 0), (64, 24), (96, 24), (128, 24), (256, 24), (128, 0)])
@pytest.mark.parametrize("cached", [True, False])
def test_a_chunk_sees_a_key_held_as_nan_at_every_place_of_a_block(ctx, D, window, cached):
    """Sixteen sequences with the key at one place of the block each, and a clean one: the rows that see it are NaN,
    the others as if it were not there."""
    import b200attn
    B, L, T = 17, 60, 64
    c = Case(ctx=[L] * B, T=T, Hq=2, Hkv=1, D=D, page=32, dtype=oracle.BF16, rope=None, window=window, seed=D + window)
    at = (40 if cached else L + 4) + np.arange(16)
    for b in range(16):
        if cached:
            _hold_nan(c, b, at[b], "k")
        else:
            c.k[b, at[b] - L, 0, 33] = np.nan
    t = c.device()
    b200attn.kv4_decode(ctx, t["q"], t["k"], t["v"], t["pages"], t["table"], t["ctx"], t["o"], c.scale, window=window,
                        **c.more())
    if cached:
        ctx.check_device_status()  # it was reported when it was stored
    else:
        with pytest.raises(b200attn.B200RuntimeException, match="4-bit cache's range"):
            ctx.check_device_status()
        for b in range(16):
            c.k[b, at[b] - L, 0, 32:64] = 0.0
    o, tol, _, _ = c.expect()
    pos = L + np.arange(T)
    sees = np.zeros((B, T), bool)
    sees[:16] = (at[:, None] <= pos) & (at[:, None] > pos - (window or 1 << 30))
    got = to_np(t["o"])
    np.testing.assert_array_equal(np.isnan(got), np.broadcast_to(sees[..., None, None], got.shape))
    assert np.all((np.abs(got - o) <= tol)[~sees])


@pytest.mark.parametrize("few,many", [
    (dict(ctx=[5000, 4100], T=2, Hq=4, Hkv=1, D=256, page=64), dict(ctx=60 + np.arange(1200) % 90, Hq=1, Hkv=1, D=64)),
    (dict(ctx=[1500] * 10, T=60, Hq=72, Hkv=9, D=256, page=64), dict(ctx=20 + np.arange(2040) % 30, Hq=9, Hkv=9, D=64)),
], ids=["hundreds", "beyond_the_workspace"])
def test_a_captured_call_and_a_later_one_with_more_units(few, many):
    """The merge counters of a call must stay zero between launches whatever an earlier captured call does: few units
    with large slots (captured), then many units with small ones, in the same workspace."""
    import torch
    import b200attn
    few, many = Case(rope=None, seed=41, **few), Case(rope=None, seed=43, **many)
    a, b = few.device(), many.device()
    with b200attn.Context(0) as one:
        def run(c, t):
            t["o"].fill_(float("nan"))
            b200attn.kv4_decode(one, t["q"], t["k"], t["v"], t["pages"], t["table"], t["ctx"], t["o"], c.scale, **c.more())

        run(few, a)
        g = _capture(lambda: run(few, a))
        size = one.workspace_bytes()
        run(many, b)
        torch.cuda.synchronize()
        first_a, first_b = a["o"].clone(), b["o"].clone()
        assert bool(torch.isfinite(first_b.float()).all())
        assert one.workspace_bytes() <= size + (1 << 17)  # more counters at most: the graph's slots stayed in place
        for _ in range(2):
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(a["o"], first_a)
            run(many, b)
            torch.cuda.synchronize()
            assert torch.equal(b["o"], first_b)
        del g
        one.check_device_status()


@pytest.mark.parametrize("D,G,T", [(64, 4, 1), (64, 7, 2), (96, 3, 1), (128, 8, 1), (256, 4, 1), (256, 4, 3)])
def test_large_key_minima_against_queries_that_cancel(ctx, D, G, T):
    """Keys whose groups lie thousands from zero, each group elsewhere, and queries whose groups sum to nearly zero
    (exact in fp16, no rotation), so that a score is made of large minima times small sums.  Two fp16 words hold a
    sum to 2^-22 of itself (the second word's rounding); products and sums are fp32, with at most 2^-20 lost of what
    they are made of (16 additions by truncation, of 2^-23 each, and the scaling).  With
        ds = scale * (2^-21 sum_y |z_y sum q| + 2^-19 sum_y (|z_y sum q| + s_y sum_i |q_i| c_i))
    an output may differ by 2^-11 of itself and (2 ds + 2^-20 + 1e-5) A, A = sum_j p_j |v_j|."""
    import b200attn
    L = 40
    c = Case(ctx=[L, 25], T=T, Hq=G, Hkv=1, D=D, rope=None, seed=D + G)
    rng = np.random.default_rng(D + G)
    q = rng.normal(size=c.q.shape).reshape(*c.q.shape[:-1], -1, 32)
    q = (q - q.mean(-1, keepdims=True)).reshape(c.q.shape)
    c.q = q.astype(np.float16).astype(np.float32)
    ds = np.zeros((2, T, G))
    for b in range(2):
        n = int(c.ctx[b])
        far = 2000.0 * rng.normal(size=(n, 1, D // 32, 1))
        k = (far + 0.3 * rng.normal(size=(n, 1, D // 32, 32))).reshape(n, 1, D).astype(np.float32)
        kc, ks = kv.quantise(k)
        vc, vs = kv.quantise(c.rows[b][1].astype(np.float32))
        c.rows[b] = [kv.values(kc, ks), kv.values(vc, vs)]
        c._store(b, 0, (kc, ks, vc, vs))
        qg = c.q[b].astype(np.float64).reshape(T, G, D // 32, 32)
        sums = np.abs(qg.sum(-1))[:, :, None]                                     # [T, G, 1, groups]
        low = np.abs(ks[:, 0, :, 1].astype(np.float64)) * sums                    # [T, G, n, groups]
        codes = np.einsum("tgyi,nyi->tgny", np.abs(qg), kc.reshape(n, -1, 32).astype(np.float64)) * ks[:, 0, :, 0].astype(np.float64)
        ds[b] = c.scale * (2.0 ** -21 * low.sum(-1) + 2.0 ** -19 * (low + codes).sum(-1)).max(-1)
    t = c.device()
    b200attn.kv4_decode(ctx, t["q"], t["k"], t["v"], t["pages"], t["table"], t["ctx"], t["o"], c.scale, **c.more())
    ctx.check_device_status()
    o, _, kh, vh = c.expect()
    for b in range(2):
        pos = int(c.ctx[b]) + np.arange(T)
        K, V = np.concatenate([c.rows[b][0], kh[b]]), np.concatenate([c.rows[b][1], vh[b]])
        A = kv.attend(c.q[b].astype(np.float64), K, np.abs(V), pos, 0, c.scale)
        tol = 2.0 ** -11 * np.abs(o[b]) + (2 * ds[b][..., None] + 2.0 ** -20 + 1e-5) * A
        err = np.abs(to_np(t["o"])[b] - o[b])
        assert np.all(err <= tol), (float((err / tol).max()), float(err.max()))


@pytest.mark.parametrize("T,dtype", [(1, oracle.F16), (1, oracle.BF16), (66, oracle.BF16)])
def test_the_widest_window_is_no_window(ctx, T, dtype):
    """Over a wide table at head dim 256, where the variant follows the keys in reach: the same bits."""
    import torch
    import b200attn
    c = Case(ctx=[1500 + 7 * b for b in range(16)], T=T, Hq=4, Hkv=1, D=256, page=64, dtype=dtype, rope=None, seed=T,
             extra_slots=1000)
    got = []
    for window in (0, 2 ** 31 - 1):
        t = c.device()
        b200attn.kv4_decode(ctx, t["q"], t["k"], t["v"], t["pages"], t["table"], t["ctx"], t["o"], c.scale,
                            window=window, **c.more())
        ctx.check_device_status()
        got.append(t["o"])
    o, tol, _, _ = c.expect()
    c.check_out(to_np(got[0]), o, tol)
    assert torch.equal(got[0], got[1])
