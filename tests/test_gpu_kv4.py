"""The paged 4-bit KV cache (b2a_kv4_append / b2a_kv4_attention / b2a_kv4_decode) against the plain
64-bit model in kv4_helpers.

Tolerances.  Stored bytes: equal (the codes are decided on 32-bit values with every operation rounded;
where a double sine or cosine enters, one code in 1e4 may fall on the other side of a rounding and a
param one fp16 step aside).  Outputs: q, k, v and the probabilities may each be rounded once to 11
significant bits and the result once to its type, so with A = sum_j p_j |v_j| and
ds = 2 * 2^-11 * scale * max_j sum_i |q_i k_ij| (two roundings in a score),
    |got - want| <= u |want| + (2 ds + 4 * 2^-11 + 1e-5) A,      u = 2^-11 (fp16), 2^-8 (bf16)
element by element, and 2e-3 (fp16) or 4e-3 (bf16) in the 2-norm, where roundings average out."""
import math

import numpy as np
import pytest

import kv4_helpers as kv
import oracle
from helpers import normal, to_dev, to_np

pytestmark = pytest.mark.gpu

UNIT = {oracle.F16: 2.0 ** -11, oracle.BF16: 2.0 ** -8}
REL = {oracle.F16: 2e-3, oracle.BF16: 4e-3}


class Case:
    """A cache with `ctx` rows already in it, T new rows (new[b] of them there) and their queries."""

    def __init__(self, *, ctx, T=1, new=None, Hq=4, Hkv=2, D=64, page=32, dtype=oracle.F16, rope="neox", theta=1e5,
                 norm=False, window=0, seed=1, extra_slots=1, stale=0xFF):
        self.ctx, self.T, self.Hq, self.Hkv, self.D, self.page = np.asarray(ctx, np.int32), T, Hq, Hkv, D, page
        self.B = B = len(ctx)
        self.new = np.full(B, T, np.int32) if new is None else np.asarray(new, np.int32)
        self.dtype, self.rope, self.theta, self.window = dtype, rope, theta, window
        self.scale = float(np.float32(1.0 / math.sqrt(D)))
        rng = np.random.default_rng(seed)
        used = -(-(self.ctx + self.new) // page)
        self.table = np.full((B, int(used.max()) + extra_slots), -1, np.int32)
        n = int(used.sum())
        ids = rng.permutation(n + 3)[:n]
        for b in range(B):
            self.table[b, :used[b]] = ids[used[:b].sum():used[:b + 1].sum()]
        self.pages = np.full((n + 3, Hkv, page * D * 5 // 4), stale, np.uint8)  # stale params: NaN
        self.rows = []  # (K, V) held, per sequence, 64-bit
        for b in range(B):
            L = int(self.ctx[b])
            k = normal(seed + 10 * b, (L, Hkv, D), oracle.F32) * np.exp(0.5 * normal(seed, (1, Hkv, D), oracle.F32))
            v = normal(seed + 10 * b + 1, (L, Hkv, D), oracle.F32)
            held = []
            codes = []
            for x in (k, v):
                c, sz = kv.quantise(x)
                held.append(kv.values(c, sz))
                codes += [c, sz]
            self.rows.append(held)
            self._store(b, 0, codes)
        self.q = normal(seed + 2, (B, T, Hq, D), dtype)
        self.k = normal(seed + 3, (B, T, Hkv, D), dtype)
        self.v = normal(seed + 4, (B, T, Hkv, D), dtype)
        self.qw = self.kw = None
        if norm:
            self.qw = (0.3 * normal(seed + 5, (D,), oracle.F32)).astype(np.float32)
            self.kw = (0.3 * normal(seed + 6, (D,), oracle.F32)).astype(np.float32)

    def _store(self, b, start, codes):
        """Rows from position `start` on, into the pages."""
        n, P = codes[0].shape[0], self.page
        for slot in range(start // P, -(-(start + n) // P)):
            lo, hi = max(start, slot * P), min(start + n, (slot + 1) * P)
            if lo >= hi:
                continue
            page = self.table[b, slot]
            got = kv.unpack(self.pages[page], self.D)
            for dst, src in zip(got, codes):  # [Hkv, P, ...] <- [n, Hkv, ...]
                dst[:, lo - slot * P:hi - slot * P] = np.swapaxes(src[lo - start:hi - start], 0, 1)
            self.pages[page] = kv.pack(*got)

    def expect(self):
        """After the call: pages, held rows, outputs, and the outputs' tolerance."""
        B, T = self.B, self.T
        o, tol = np.zeros((B, T, self.Hq, self.D)), np.zeros((B, T, self.Hq, self.D))
        kh, vh = np.zeros(self.k.shape), np.zeros(self.k.shape)
        for b in range(B):
            n, L = int(self.new[b]), int(self.ctx[b])
            if n == 0:
                continue
            pos = L + np.arange(n)
            kc, ks = kv.quantise(kv.norm_rope(self.k[b, :n], self.kw, pos, self.rope, self.theta))
            vc, vs = kv.quantise(self.v[b, :n])
            self._store(b, L, (kc, ks, vc, vs))
            kh[b, :n], vh[b, :n] = kv.values(kc, ks), kv.values(vc, vs)
            K = np.concatenate([self.rows[b][0], kh[b, :n]])
            V = np.concatenate([self.rows[b][1], vh[b, :n]])
            q = kv.norm_rope(self.q[b, :n], self.qw, pos, self.rope, self.theta, bits=64)
            o[b, :n] = kv.attend(q, K, V, pos, self.window, self.scale)
            A = kv.attend(q, K, np.abs(V), pos, self.window, self.scale)
            G = self.Hq // self.Hkv
            top = np.max(np.einsum("thd,mhd->thm", np.abs(q), np.repeat(np.abs(K), G, 1)), -1)
            ds = 2 * 2.0 ** -11 * self.scale * top
            tol[b, :n] = UNIT[self.dtype] * np.abs(o[b, :n]) + (2 * ds[..., None] + 4 * 2.0 ** -11 + 1e-5) * A
        return o, tol, kh, vh

    def device(self):
        import torch
        t = {n: to_dev(getattr(self, n), self.dtype) for n in ("q", "k", "v")}
        t.update(pages=torch.from_numpy(self.pages.copy()).cuda(), table=torch.from_numpy(self.table).cuda(),
                 ctx=torch.from_numpy(self.ctx).cuda(), new=torch.from_numpy(self.new).cuda(),
                 qw=None if self.qw is None else torch.from_numpy(self.qw).cuda(),
                 kw=None if self.kw is None else torch.from_numpy(self.kw).cuda())
        t["o"] = torch.full_like(t["q"], float("nan"))
        t["k_held"], t["v_held"] = torch.full_like(t["k"], float("nan")), torch.full_like(t["v"], float("nan"))
        return t

    def more(self):
        import b200attn
        mode = {None: b200attn.ROPE_NONE, "neox": b200attn.ROPE_NEOX, "gemma": b200attn.ROPE_GEMMA}[self.rope]
        return dict(rope_mode=mode, rope_theta=self.theta)

    def check_pages(self, got, exact):
        g, w = kv.unpack(got, self.D), kv.unpack(self.pages, self.D)
        if exact:
            np.testing.assert_array_equal(got, self.pages)
            return
        for i in (0, 2):
            diff = g[i] != w[i]
            assert diff.mean() <= 1e-4 and np.abs(g[i].astype(int) - w[i]).max() <= 1
        for i in (1, 3):
            a, b = g[i].view(np.uint16).astype(int), w[i].view(np.uint16).astype(int)
            assert np.abs(a - b).max() <= 1 and (a != b).mean() <= 1e-4

    def check_out(self, got, o, tol):
        assert np.all(np.isfinite(got))
        err = np.abs(got - o)
        assert np.all(err <= tol), (float((err - tol).max()), float(err.max()))
        if np.linalg.norm(o):
            rel = np.linalg.norm(got - o) / np.linalg.norm(o)
            assert rel <= REL[self.dtype], rel

    def run_decode(self, ctx, **kw):
        import b200attn
        t = self.device()
        b200attn.kv4_decode(ctx, t["q"], t["k"], t["v"], t["pages"], t["table"], t["ctx"], t["o"], self.scale,
                            new_lens=t["new"], window=self.window, q_norm_w=t["qw"], k_norm_w=t["kw"],
                            k_held=t["k_held"], v_held=t["v_held"], **self.more(), **kw)
        ctx.check_device_status()
        o, tol, kh, vh = self.expect()
        self.check_pages(t["pages"].cpu().numpy(), exact=self.rope is None and self.kw is None)
        self.check_out(to_np(t["o"]), o, tol)
        u = UNIT[self.dtype]
        np.testing.assert_allclose(to_np(t["v_held"]), vh, rtol=u, atol=1e-7)
        # a code on the other side of its rounding moves a key by one step: at most 1e-4 of them
        far = np.abs(to_np(t["k_held"]) - kh) > u * np.abs(kh) + 1e-6
        assert far.mean() <= 1e-4
        return t


CASES = {
    "one_key": dict(ctx=[0]),
    "first_block": dict(ctx=[1, 15, 16, 17], D=64),
    "page_edges": dict(ctx=[31, 32, 33, 63, 64, 95, 96, 100]),
    "qwen": dict(ctx=[500, 1, 259, 700], Hq=14, Hkv=2, D=64, theta=1e6, dtype=oracle.BF16),
    "long_split": dict(ctx=[9001, 2], Hq=7, Hkv=1, D=64, page=64, theta=1e6),
    "mha_96": dict(ctx=[100, 0, 259], Hq=4, Hkv=4, D=96, page=48),
    "gqa_128": dict(ctx=[10, 399, 200], Hq=8, Hkv=2, D=128, page=16, dtype=oracle.BF16),
    "sixteen_heads": dict(ctx=[150, 299], Hq=16, Hkv=1, D=128, page=128),
    "odd_heads": dict(ctx=[77, 130], Hq=15, Hkv=3, D=64, page=80),
    "forty_heads_each": dict(ctx=[70, 33], Hq=40, Hkv=1, D=64),
    "gemma_local": dict(ctx=[0, 19, 20, 21, 300, 640], Hq=4, Hkv=1, D=256, page=64, rope="gemma", theta=1e4, norm=True,
                        window=20),
    "gemma_global": dict(ctx=[700, 40], Hq=4, Hkv=1, D=256, page=256, rope="gemma", theta=1e6, norm=True,
                         dtype=oracle.BF16),
    "window_one": dict(ctx=[0, 5, 64], window=1),
    "no_rope": dict(ctx=[3, 40, 81], rope=None),
    "many_sequences": dict(ctx=list(range(0, 330)), Hq=2, Hkv=1, D=64, page=16),
    "verify": dict(ctx=[0, 30, 61, 300], T=5, Hq=9, Hkv=3, D=64, page=48, dtype=oracle.BF16),
    "verify_ragged": dict(ctx=[0, 30, 61, 300, 7], T=6, new=[6, 0, 1, 5, 3], Hq=4, Hkv=4, D=96),
    "all_idle": dict(ctx=[0, 30], T=3, new=[0, 0], D=64),
    "verify_window": dict(ctx=[0, 30, 100], T=7, Hq=8, Hkv=1, D=256, window=10, rope="gemma", norm=True),
    "chunk": dict(ctx=[100, 0], T=70, Hq=4, Hkv=2, D=128, page=64),
    "chunk_ragged": dict(ctx=[33, 0, 411], T=150, new=[150, 17, 97], Hq=8, Hkv=1, D=64, dtype=oracle.BF16),
    "chunk_window": dict(ctx=[200], T=140, Hq=4, Hkv=1, D=256, window=50, rope="gemma", norm=True, page=48),
    "chunk_mha_96": dict(ctx=[65, 130], T=200, Hq=2, Hkv=2, D=96, page=16),
    "chunk_bf16_128": dict(ctx=[100, 0, 1000], T=64, Hq=4, Hkv=2, D=128, page=64, dtype=oracle.BF16),
    "chunk_bf16_window": dict(ctx=[200, 10], T=140, Hq=4, Hkv=1, D=256, window=50, rope="gemma", norm=True, page=48,
                              dtype=oracle.BF16),
    "chunk_bf16_96": dict(ctx=[65, 130, 0], T=300, new=[300, 0, 129], Hq=2, Hkv=2, D=96, page=16, dtype=oracle.BF16),
    "chunk_bf16_wide_window": dict(ctx=[700, 0, 300], T=257, new=[257, 256, 1], Hq=3, Hkv=1, D=64, window=300, page=80,
                                   rope=None, dtype=oracle.BF16),
    "chunk_prompt": dict(ctx=[0], T=300, Hq=4, Hkv=2, D=64, rope=None),
}


@pytest.mark.parametrize("name", list(CASES))
def test_decode_matches_the_model(ctx, name):
    Case(seed=sum(map(ord, name)), **CASES[name]).run_decode(ctx)


@pytest.mark.parametrize("D,dtype,rope,norm", [(64, oracle.F16, None, False), (96, oracle.BF16, "neox", True),
                                               (128, oracle.F16, "gemma", False), (256, oracle.BF16, "neox", True),
                                               (128, oracle.BF16, None, False)])
def test_append_stores_the_definition(ctx, D, dtype, rope, norm):
    """Bytes of every touched row; every other byte (stale ones too) as it was; ragged and absent rows."""
    import b200attn
    c = Case(ctx=[0, 5, 47, 16, 300], T=37, new=[37, 0, 37, 16, 1], Hq=2, Hkv=2, D=D, page=48, dtype=dtype, rope=rope,
             norm=norm, seed=D, stale=0xA5)
    t = c.device()
    b200attn.kv4_append(ctx, t["k"], t["v"], t["pages"], t["table"], t["ctx"], new_lens=t["new"], k_norm_w=t["kw"],
                        k_held=t["k_held"], v_held=t["v_held"], **c.more())
    ctx.check_device_status()
    _, _, kh, vh = c.expect()
    c.check_pages(t["pages"].cpu().numpy(), exact=rope is None and not norm)
    np.testing.assert_allclose(to_np(t["v_held"]), vh, rtol=UNIT[dtype], atol=1e-7)
    assert (np.abs(to_np(t["k_held"]) - kh) > UNIT[dtype] * np.abs(kh) + 1e-6).mean() <= 1e-4


def test_append_special_rows(ctx):
    """Constant groups (s = 0), tiny ranges (fp16 subnormal s), large ones, both zeros; then values that are
    not finite or beyond fp16: their group alone holds NaN and the device status says so."""
    import torch
    import b200attn
    c = Case(ctx=[0], T=6, Hq=2, Hkv=2, D=64, rope=None, dtype=oracle.BF16)
    c.k[0, 0] = 0.0
    c.k[0, 1, :, :32], c.k[0, 1, :, 32:] = 3.0, -0.0
    c.k[0, 2] *= 2.0 ** -20
    c.v[0, 3] *= 2.0 ** 13
    c.k, c.v = (oracle.round_to(x, oracle.BF16).reshape(x.shape) for x in (c.k, c.v))
    c.run_decode(ctx)
    c = Case(ctx=[0], T=4, Hq=2, Hkv=2, D=64, rope=None, dtype=oracle.BF16)
    c.k[0, 0, 0, 3] = np.inf
    c.v[0, 1, 1, 40] = np.nan
    c.k[0, 2, 1, 0] = 1e6
    t = c.device()
    b200attn.kv4_append(ctx, t["k"], t["v"], t["pages"], t["table"], t["ctx"], k_held=t["k_held"], v_held=t["v_held"],
                        **c.more())
    with pytest.raises(b200attn.B200RuntimeException) as ei:
        ctx.check_device_status()
    assert ei.value.status == b200attn.B2A_EDEVICE and "4-bit cache's range" in str(ei.value)
    ctx.check_device_status()  # reported once
    _, _, kh, vh = c.expect()
    g = kv.unpack(t["pages"].cpu().numpy(), 64)
    w = kv.unpack(c.pages, 64)
    for a, b in zip(g, w):
        np.testing.assert_array_equal(np.nan_to_num(a.astype(np.float64), nan=-1), np.nan_to_num(b.astype(np.float64), nan=-1))
    np.testing.assert_array_equal(np.isnan(to_np(t["k_held"])), np.isnan(kh))
    np.testing.assert_array_equal(np.isnan(to_np(t["v_held"])), np.isnan(vh))


def test_fused_rows_strides_and_side_stream(ctx):
    """q, k and v as slices of one fused [Q|K|V] projection, on a stream that is not the current one."""
    import torch
    import b200attn
    c = Case(ctx=[20, 0, 77], T=3, Hq=4, Hkv=2, D=64, seed=8)
    t = c.device()
    B, T, Hq, Hkv, D = c.B, c.T, c.Hq, c.Hkv, c.D
    fused = torch.cat([t[n].reshape(B, T, -1) for n in ("q", "k", "v")], -1).contiguous()
    q, k, v = (x.unflatten(-1, (-1, D)) for x in fused.split([Hq * D, Hkv * D, Hkv * D], -1))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    b200attn.kv4_decode(ctx, q, k, v, t["pages"], t["table"], t["ctx"], t["o"], c.scale, stream=side, **c.more())
    ctx.check_device_status(side)
    o, tol, _, _ = c.expect()
    c.check_out(to_np(t["o"]), o, tol)
    # one token each, rows of a longer array
    c = Case(ctx=[20, 0, 77], Hq=4, Hkv=2, D=64, seed=9)
    t = c.device()
    wide = torch.zeros(c.B, 5, (Hq + 2 * Hkv), D, dtype=torch.float16, device="cuda")
    wide[:, 2] = torch.cat([t["q"][:, 0], t["k"][:, 0], t["v"][:, 0]], 1)
    q, k, v = wide[:, 2:3].split([Hq, Hkv, Hkv], 2)
    b200attn.kv4_decode(ctx, q, k, v, t["pages"], t["table"], t["ctx"], t["o"], c.scale, **c.more())
    ctx.check_device_status()
    o, tol, _, _ = c.expect()
    c.check_out(to_np(t["o"]), o, tol)


def test_more_sequences_than_one_launch_takes(ctx):
    """2100 short sequences, one and several tokens each: the call runs in two slices."""
    lens = np.arange(2100) % 37
    Case(ctx=lens, Hq=2, Hkv=1, D=64, page=16, seed=3, rope=None).run_decode(ctx)
    Case(ctx=lens, T=2, new=(np.arange(2100) % 3), Hq=1, Hkv=1, D=64, page=16, seed=5, dtype=oracle.BF16).run_decode(ctx)


def test_slices_of_a_call_share_their_variant(ctx):
    """At head dim 256 the kernel's variant follows the whole call's work, of which the last slice has
    little."""
    lens = np.arange(2100) % 29
    lens[2090] = 330
    Case(ctx=lens, Hq=2, Hkv=1, D=256, page=16, seed=4, rope=None, dtype=oracle.BF16).run_decode(ctx)
    Case(ctx=lens, Hq=1, Hkv=1, D=256, page=16, seed=7, rope=None).run_decode(ctx)


def test_pages_beyond_four_gigabytes(ctx):
    """The pages in use lie past 2^32 bytes of their pool."""
    import torch
    for T, dtype in ((3, oracle.F16), (70, oracle.BF16)):
        c = Case(ctx=[1500, 40], T=T, Hq=4, Hkv=2, D=64, page=64, seed=6, dtype=dtype)
        t = c.device()
        page_bytes = c.pages[0].size
        first = (1 << 32) // page_bytes + 5
        big = torch.empty((first + c.pages.shape[0], 2, 64 * 80), dtype=torch.uint8, device="cuda")
        big[first:] = t["pages"]
        t["table"] = torch.where(t["table"] >= 0, t["table"] + first, t["table"])
        import b200attn
        b200attn.kv4_decode(ctx, t["q"], t["k"], t["v"], big, t["table"], t["ctx"], t["o"], c.scale, **c.more())
        ctx.check_device_status()
        o, tol, _, _ = c.expect()
        c.check_out(to_np(t["o"]), o, tol)
        c.check_pages(big[first:].cpu().numpy(), exact=False)
        del big


@pytest.mark.parametrize("T", [1, 5, 80])
def test_graph_replays_recompute_the_step(ctx, T):
    import torch
    import b200attn
    c = Case(ctx=[700, 3, 90], T=T, Hq=4, Hkv=2, D=128, dtype=oracle.BF16, seed=T)
    t = c.device()
    run = lambda: b200attn.kv4_decode(ctx, t["q"], t["k"], t["v"], t["pages"], t["table"], t["ctx"], t["o"], c.scale, **c.more())
    run()  # workspaces reach their final size before capture
    torch.cuda.synchronize()
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    o, tol, _, _ = c.expect()
    for _ in range(3):
        t["o"].fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        c.check_out(to_np(t["o"]), o, tol)
    del g
    ctx.check_device_status()


def test_workspace_limit_and_its_fallback():
    """A cap below the decode workspace is B2A_EOOM; one that only leaves no room for a chunk's staged
    rows makes the chunk read the codes instead."""
    import b200attn
    c = Case(ctx=[300, 20], T=2, Hq=4, Hkv=2, D=64, seed=2)
    t = c.device()
    with b200attn.Context(0) as small:
        small.set_workspace_limit(4096)
        with pytest.raises(b200attn.B200RuntimeException) as ei:
            b200attn.kv4_decode(small, t["q"], t["k"], t["v"], t["pages"], t["table"], t["ctx"], t["o"], c.scale, **c.more())
        assert ei.value.status == b200attn.B2A_EOOM and "exceeds the context limit" in str(ei.value)
        assert small.workspace_bytes() <= 4096
        small.set_workspace_limit(0)
        c.run_decode(small)
    c = Case(ctx=[5000, 20], T=70, Hq=2, Hkv=1, D=64, seed=2, dtype=oracle.BF16, extra_slots=20000)
    with b200attn.Context(0) as small:
        small.set_workspace_limit(30 << 20)
        c.run_decode(small)
        assert small.workspace_bytes() <= 30 << 20


def test_attention_alone_and_repeated_calls_agree(ctx):
    """kv4_attention after kv4_append gives kv4_decode's outputs; the same call twice gives the same bits."""
    import torch
    import b200attn
    c = Case(ctx=[400, 3, 1200], T=4, Hq=7, Hkv=1, D=128, seed=4)
    t = c.run_decode(ctx)
    first = t["o"].clone()
    for _ in range(3):
        t["o"].fill_(float("nan"))
        b200attn.kv4_attention(ctx, t["q"], t["pages"], t["table"], t["ctx"], t["o"], c.scale, new_lens=t["new"],
                               **c.more())
        ctx.check_device_status()
        o, tol, _, _ = c.expect()
        c.check_out(to_np(t["o"]), o, tol)
        again = t["o"].clone()
        b200attn.kv4_attention(ctx, t["q"], t["pages"], t["table"], t["ctx"], t["o"], c.scale, new_lens=t["new"],
                               **c.more())
        assert torch.equal(again, t["o"])
    b200attn.kv4_decode(ctx, t["q"], t["k"], t["v"], t["pages"], t["table"], t["ctx"], t["o"], c.scale, **c.more())
    assert torch.equal(first, t["o"])


def test_large_scores_and_values(ctx):
    """Scores in the hundreds (the running maximum moves), values near fp16's limit beside tiny ones."""
    c = Case(ctx=[130, 700], Hq=4, Hkv=2, D=64, rope=None, dtype=oracle.BF16, seed=12)
    c.q *= 32.0
    for b in range(c.B):
        for h, f in ((0, 3000.0), (1, 2.0 ** -12)):
            x = c.rows[b][1][:, h] * f
            code, sz = kv.quantise(x.astype(np.float32))
            kc, ks = kv.quantise(c.rows[b][0].astype(np.float32))
            c.rows[b][1][:, h] = kv.values(code, sz)
            full = kv.quantise(c.rows[b][1].astype(np.float32))
            c.rows[b] = [kv.values(kc, ks), kv.values(*full)]
            c._store(b, 0, (kc, ks, *full))
    c.run_decode(ctx)


@pytest.mark.parametrize("T", [2, 70])
def test_bad_lengths_and_pages_are_reported_and_contained(ctx, T):
    import torch
    import b200attn
    c = Case(ctx=[20, 40, 50], T=T, Hq=4, Hkv=2, D=64, seed=5, extra_slots=0, dtype=oracle.BF16)
    t = c.device()
    t["ctx"][1] = 10 ** 6
    before = t["pages"].clone()
    b200attn.kv4_decode(ctx, t["q"], t["k"], t["v"], t["pages"], t["table"], t["ctx"], t["o"], c.scale, **c.more())
    with pytest.raises(b200attn.B200RuntimeException) as ei:
        ctx.check_device_status()
    assert ei.value.status == b200attn.B2A_EDEVICE and "ctx_lens" in str(ei.value)
    assert bool(torch.isnan(t["o"][1]).all()) and bool(torch.isfinite(t["o"][[0, 2]].float()).all())
    mine = torch.from_numpy(c.table[1]).cuda().long()
    assert torch.equal(t["pages"][mine], before[mine])
    for bad in (-1, 10 ** 6):
        t = c.device()
        t["table"][2, 0] = bad
        b200attn.kv4_decode(ctx, t["q"], t["k"], t["v"], t["pages"], t["table"], t["ctx"], t["o"], c.scale, **c.more())
        with pytest.raises(b200attn.B200RuntimeException) as ei:
            ctx.check_device_status()
        assert ei.value.status == b200attn.B2A_EDEVICE and "page_table" in str(ei.value)
        assert bool(torch.isnan(t["o"][2]).all()) and bool(torch.isfinite(t["o"][:2].float()).all())
    ctx.check_device_status()


def test_refusals(ctx):
    import torch
    import b200attn
    c = Case(ctx=[20, 40], T=2, Hq=4, Hkv=2, D=64)
    t = c.device()

    def call(**kw):
        a = {**t, **kw}
        b200attn.kv4_decode(ctx, a["q"], a["k"], a["v"], a["pages"], a["table"], a["ctx"], a["o"], a.get("scale", c.scale),
                            new_lens=a["new"], window=a.get("window", 0), q_norm_w=a["qw"], k_norm_w=a["kw"],
                            rope_mode=a.get("rope_mode", 1), rope_theta=a.get("rope_theta", 1e4))

    w = torch.ones(64, device="cuda")
    for bad, what in ((dict(q=t["q"][:, :, :3]), "o expected shape"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
                      (dict(window=-1), "window"), (dict(rope_mode=7), "rope mode"), (dict(rope_theta=0.0), "theta"),
                      (dict(qw=w), "together"), (dict(qw=w[:32], kw=w), "float32"), (dict(ctx=t["ctx"].long()), "int32"),
                      (dict(new=t["new"][:1]), "int32"), (dict(table=t["table"][:1]), "page_table"),
                      (dict(pages=t["pages"].int()), "uint8"), (dict(pages=t["pages"][:, :1].contiguous()), "kv heads"),
                      (dict(pages=t["pages"][:, :, :-16].contiguous()), "no whole rows"),
                      (dict(k=t["k"].bfloat16()), "element type"), (dict(o=t["o"].float()), "element type"),
                      (dict(k=t["k"].cpu()), "CUDA device"), (dict(k=t["k"].transpose(1, 2).contiguous().transpose(1, 2)), "strides"),
                      (dict(pages=t["pages"].cpu()), "CUDA device")):
        with pytest.raises(ValueError, match=what):
            call(**bad)
    o3 = torch.empty(2, 2, 3, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="divisible"):
        call(q=t["q"][:, :, :3].contiguous(), o=o3)
    f = {n: t[n].float() for n in ("q", "k", "v", "o")}
    with pytest.raises(b200attn.B200RuntimeException) as ei:
        call(**f)
    assert ei.value.status == b200attn.B2A_ENOTSUP
    z = torch.zeros(2, 2, 2, 32, dtype=torch.float16, device="cuda")
    with pytest.raises(b200attn.B200RuntimeException) as ei:
        b200attn.kv4_append(ctx, z, z, torch.zeros(4, 2, 16 * 40, dtype=torch.uint8, device="cuda"), t["table"], t["ctx"])
    assert ei.value.status == b200attn.B2A_ENOTSUP
    ctx.check_device_status()


@pytest.mark.parametrize("T", [30, 66])
@pytest.mark.parametrize("D,Hq,dtype", [(64, 4, oracle.F16), (64, 7, oracle.F16), (96, 5, oracle.BF16), (128, 12, oracle.BF16),
                                        (256, 4, oracle.F16), (256, 6, oracle.F16), (256, 3, oracle.BF16)])
def test_a_key_held_as_nan_reaches_only_the_rows_that_see_it(ctx, D, Hq, dtype, T):
    """A value group or a key group that is held as NaN: the rows before it are untouched; the rows that see it
    are NaN, in that group alone (value) or whole (key); with a window it leaves sight again."""
    import torch
    import b200attn
    for which, window in (("v", 0), ("k", 0), ("v", 20), ("k", 20)):
        c = Case(ctx=[45, 8], T=T, Hq=Hq, Hkv=1, D=D, rope=None, dtype=dtype, window=window, seed=D + Hq)
        x = c.k if which == "k" else c.v
        x[0, 4, 0, 33] = np.nan
        t = c.device()
        b200attn.kv4_decode(ctx, t["q"], t["k"], t["v"], t["pages"], t["table"], t["ctx"], t["o"], c.scale,
                            window=window, **c.more())
        with pytest.raises(b200attn.B200RuntimeException):
            ctx.check_device_status()
        x[0, 4, 0, 32:64] = 0.0  # the model without it, for the rows that do not see it
        x[0, 4, 0, 33] = 0.0
        o, tol, _, _ = c.expect()
        got = to_np(t["o"])
        sees = np.zeros((2, T), bool)
        sees[0, 4:(24 if window else T)] = True
        bad = np.zeros(got.shape, bool)
        bad[sees] = True
        if which == "v":
            bad[..., :32] = False
            bad[..., 64:] = False
        np.testing.assert_array_equal(np.isnan(got), bad, err_msg=f"{which} window {window}")
        if which == "v":  # other groups of the rows that see it are as if it were a number
            ok = ~bad
        else:
            ok = np.broadcast_to(~sees[..., None, None], got.shape)
        assert np.all(np.abs(got - o)[ok] <= tol[ok])
