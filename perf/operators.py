"""The operators of the paged 4-bit KV cache, with their plain forms: appending rows (b2a_kv4_append), attending
over the cache (b2a_kv4_decode) and managing its pages (b2a_pages_reserve / fork / free / compact).

Cache.  A layer's pool is uint8 [num_pages][Hkv][page_size * D * 5 / 4]; page_table int32 [B][max_pages] names the
page that holds positions [i * page_size, (i + 1) * page_size) of sequence b (-1: none).  A (page, head) slab is a
row of blocks of 16 keys, each [K codes][K params][V codes][V params].  A row of D values is held in groups of 32:
    lo, hi = min, max of the group;  s = f16((hi - lo) * f32(1/15));  z = f16(lo)
    c = clamp(rint((x - z) * (1 / s)), 0, 15), every operation in 32 bits;  c = 0 where s = 0
    value held = s * c + z
so the codes are whole numbers decided on 32-bit values.  Place of a code in its block (key 0..15, d = 32 y + r):
    K: d = 32 y + 16 x + 8 j + 2 t + e, key = g + 8 r       V: key = 2 t + e + 8 r, d = 32 y + 16 x + 8 j + g
    byte ((y * 8 + g) * 4 + t) * 8 + x * 4 + 2 e + r, low nibble j = 0, high nibble j = 1
and of the pair (s, z) of key g + 8 r, group y: half2 number (g * 2 + r) * (D / 32) + y.

Attention.  Query t of sequence b sits at p = ctx_lens[b] + t and sees keys [max(0, p - window + 1), p] (window 0: from
0), the new rows as the cache holds them; rows t >= new_lens[b] do not exist: nothing is stored, outputs are zero.
"""
import math

import torch

own = False

GROUP = 32
FIFTEENTH = float(torch.tensor(1.0, dtype=torch.float32) / torch.tensor(15.0, dtype=torch.float32))
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = float(torch.tensor(1e-6, dtype=torch.float32))


def listed():
    return [
        # one user's single token in a short chat: a Qwen2.5-0.5B layer, where only latency counts
        dict(name="decode_one", op="decode", B=1, T=1, Hq=14, Hkv=2, D=64, lo=500, hi=500, ragged=False, page=32,
             window=0, rope="neox", theta=1e6, norm=False, type="bf16"),
        # the repository's batched decode workload (64 sequences, contexts 512..8192) on a 4-bit cache
        dict(name="decode_batch", op="decode", B=64, T=1, Hq=14, Hkv=2, D=64, lo=512, hi=8192, ragged=False, page=64,
             window=0, rope="neox", theta=1e6, norm=False, type="fp16"),
        # a Gemma-3 sliding-window layer: QK-norm, window 512, contexts far longer than the window
        dict(name="decode_local", op="decode", B=256, T=1, Hq=4, Hkv=1, D=256, lo=1024, hi=32768, ragged=False, page=64,
             window=512, rope="gemma", theta=1e4, norm=True, type="fp16"),
        # the same model's global layer over the whole contexts: the largest cache
        dict(name="decode_global", op="decode", B=256, T=1, Hq=4, Hkv=1, D=256, lo=1024, hi=32768, ragged=False,
             page=64, window=0, rope="gemma", theta=1e6, norm=True, type="fp16"),
        # speculative verification: up to 5 draft tokens, ragged, idle slots among them, odd page size
        dict(name="verify_ragged", op="decode", B=24, T=5, Hq=9, Hkv=3, D=64, lo=0, hi=3001, ragged=True, page=48,
             window=0, rope="neox", theta=1e5, norm=False, type="bf16"),
        # a chunk of a prompt on a cached (shared) prefix: compute-bound
        dict(name="chunk_prompt", op="decode", B=2, T=1000, Hq=32, Hkv=8, D=128, lo=2000, hi=4000, ragged=False,
             page=128, window=0, rope="neox", theta=1e6, norm=False, type="bf16"),
        # storing the prompts of the repository's prefill workload (Phi-3 heads) after their prefill
        dict(name="append_prompt", op="append", B=8, T=4096, Hkv=32, D=96, lo=0, hi=0, ragged=False, page=64,
             rope="neox", theta=1e4, norm=False, type="bf16"),
        # ragged suffixes behind cached prefixes, starting and ending inside pages and blocks, with key norm
        dict(name="append_ragged", op="append", B=5, T=37, Hkv=4, D=128, lo=3, hi=700, ragged=True, page=16,
             rope="neox", theta=1e6, norm=True, type="fp16"),
        # a speculative step of a small server: drop the last draft's pages, reserve the next one's
        dict(name="draft_small", op="draft", B=8, T=6, lo=20, hi=900, page=16, layers=2, Hkv=2, D=64),
        # the same for a full batch: the page table and the reference counts are what moves
        dict(name="draft_large", op="draft", B=1024, T=9, lo=200, hi=8000, page=16, layers=1, Hkv=1, D=64),
        # one step of beam search: the rows fork from their parents, written pages are copied first
        dict(name="beam_step", op="beam", B=64, T=1, lo=100, hi=2000, beams=4, page=64, layers=4, Hkv=2, D=128),
        # continuous batching: the oldest requests leave, the pool is compacted, new ones are admitted
        dict(name="churn", op="churn", B=48, T=0, lo=900, hi=1100, leave=5, page=64, layers=4, Hkv=2, D=128),
    ]


HEADS = [(14, 2, 64), (9, 3, 64), (32, 32, 96), (4, 1, 256), (32, 8, 128), (16, 1, 128), (12, 12, 64), (40, 8, 128)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges: contexts and batches over their logarithm, head layouts of the repository's
    configurations and of common models, every page size and type."""
    kinds = {"draft": "pages", "beam": "pages", "churn": "pages"}
    top = {}  # the largest listed case of each operator: no drawn case costs more
    for c in listed():
        w, kind = work(c), kinds.get(c["op"], c["op"])
        top[kind] = tuple(max(a, b) for a, b in zip(top.get(kind, (0, 0)), (w["bytes"], w["flops"])))
    while True:
        op = rng.choice(["decode"] * 5 + ["append"] * 2 + ["draft", "beam", "churn"])
        Hq, Hkv, D = rng.choice(HEADS)
        if op in ("decode", "append"):
            T = 1 if op == "decode" and rng.random() < 0.6 else _log(rng, 1, 1024) if rng.random() < 0.5 else rng.randint(1, 16)
            hi = _log(rng, 1, 32768)
            c = dict(op=op, B=_log(rng, 1, 256), T=T, Hq=Hq, Hkv=Hkv, D=D, lo=rng.randint(0, hi), hi=hi,
                     ragged=T > 1 and rng.random() < 0.5, page=rng.choice([16, 32, 48, 64, 128, 256]),
                     window=rng.choice([0, 0, _log(rng, 16, 4096)]), rope=rng.choice(["neox", "neox", "gemma", "none"]),
                     theta=rng.choice([1e4, 1e5, 1e6]), norm=rng.random() < 0.3, type=rng.choice(["bf16", "fp16"]))
            if op == "append":
                del c["Hq"], c["window"]
        else:
            lo = _log(rng, 1, 4000)
            c = dict(op=op, B=_log(rng, 4, 1024), T=rng.randint(1, 16), lo=lo, hi=lo + rng.randint(0, 4000),
                     page=rng.choice([16, 32, 48, 64, 128]), layers=rng.randint(1, 4), Hkv=rng.choice([1, 2, 4]),
                     D=rng.choice([64, 96, 128, 256]))
            if op == "beam":
                c.update(beams=rng.randint(2, 8))
                c["B"] = max(1, c["B"] // c["beams"]) * c["beams"]
            if op == "churn":
                c.update(leave=rng.randint(1, max(1, c["B"] // 4)), T=0)
        kind, w = kinds.get(op, op), work(c)
        pool = c["B"] * (1.6 if kind == "pages" else 1) * (c["hi"] + c["T"] + c["page"]) * c.get("layers", 1) * c["Hkv"] * c["D"] * 1.25
        if w["bytes"] <= top[kind][0] and w["flops"] <= top[kind][1] and pool < (1e9 if kind == "pages" else 3e9):
            return c


# ------------------------------------------------------------------ the cache's layout
def _pack(kc, ks, kz, vc, vs, vz):
    """Codes [..., 16 keys, D] and params [..., 16, D/32] of whole blocks -> bytes [..., 20 D]."""
    head, D = kc.shape[:-2], kc.shape[-1]
    n, y = len(head), D // GROUP
    # K: key -> (r, g), d -> (y, x, j, t, e);  V: key -> (r, t, e), d -> (y, x, j, g);  both -> (y, g, t, x, e, r | j)
    k = kc.reshape(*head, 2, 8, y, 2, 2, 4, 2).permute(*range(n), *(n + i for i in (2, 1, 5, 3, 6, 0, 4)))
    v = vc.reshape(*head, 2, 4, 2, y, 2, 2, 8).permute(*range(n), *(n + i for i in (3, 6, 1, 4, 2, 0, 5)))
    kb = (k[..., 0] | (k[..., 1] << 4)).reshape(*head, 8 * D)
    vb = (v[..., 0] | (v[..., 1] << 4)).reshape(*head, 8 * D)

    def params(s, z):
        p = torch.stack([s, z], -1).reshape(*head, 2, 8, y, 2).transpose(n, n + 1).contiguous()
        return p.view(torch.uint8).reshape(*head, 2 * D)

    return torch.cat([kb, params(ks, kz), vb, params(vs, vz)], -1)


def _unpack(blocks, D):
    """Bytes [..., 20 D] of whole blocks -> values held in 32 bits, K and V [..., 16, D]."""
    head = blocks.shape[:-1]
    n, y = len(head), D // GROUP

    def nibbles(b):
        return torch.stack([b & 15, b >> 4], -1).reshape(*head, y, 8, 4, 2, 2, 2, 2)  # (y, g, t, x, e, r, j)

    def params(b):
        p = b.contiguous().view(torch.float16).reshape(*head, 8, 2, y, 2).transpose(n, n + 1)
        return p.reshape(*head, 16, y, 1, 2).float()

    k = nibbles(blocks[..., :8 * D]).permute(*range(n), *(n + i for i in (5, 1, 0, 3, 6, 2, 4)))
    v = nibbles(blocks[..., 10 * D:18 * D]).permute(*range(n), *(n + i for i in (5, 2, 4, 0, 3, 6, 1)))
    kp, vp = params(blocks[..., 8 * D:10 * D]), params(blocks[..., 18 * D:])
    k = k.reshape(*head, 16, y, GROUP).float().mul_(kp[..., 0]).add_(kp[..., 1])
    v = v.reshape(*head, 16, y, GROUP).float().mul_(vp[..., 0]).add_(vp[..., 1])
    return k.reshape(*head, 16, D), v.reshape(*head, 16, D)


def _quantise(x):
    """Codes uint8 [..., D], params f16 [..., D/32] of 32-bit rows x [..., D]."""
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    lo, hi = g.amin(-1), g.amax(-1)
    s, z = ((hi - lo) * FIFTEENTH).half(), lo.half()
    sf = s.float()
    inv = torch.where(sf > 0, sf.reciprocal(), torch.zeros_like(sf))
    c = ((g - z.float()[..., None]) * inv[..., None]).round().clamp(0, 15)
    return c.to(torch.uint8).reshape(x.shape), s, z


def _held(c, s, z):
    g = c.reshape(*c.shape[:-1], -1, GROUP).float() * s.float()[..., None] + z.float()[..., None]
    return g.reshape(c.shape)


# ------------------------------------------------------------------ inputs
def _lens(c, g):
    lens = torch.randint(c["lo"], c["hi"] + 1, (c["B"],), device="cuda", dtype=torch.int32, generator=g)
    new = torch.full((c["B"],), c["T"], device="cuda", dtype=torch.int32)
    if c.get("ragged"):
        new = torch.randint(0, c["T"] + 1, (c["B"],), device="cuda", dtype=torch.int32, generator=g)
        new[0] = c["T"]
    return lens, new


def _table(used, g, slack=0.06):
    """A page table whose row b names used[b] pages of a pool at random places, and the pool's size."""
    B, total = used.numel(), int(used.sum())
    pool = total + max(2, int(total * slack))
    order = torch.randperm(pool, device="cuda", generator=g)[:total].int()
    slot = torch.arange(max(1, int(used.max())), device="cuda")
    at = (used.long().cumsum(0) - used)[:, None] + slot
    table = torch.where(slot < used[:, None], order[at.clamp(max=max(0, total - 1))] if total else -1, -1)
    return table.int().contiguous(), pool


def _ceil(a, b):
    return (a + b - 1) // b


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    if c["op"] in ("draft", "beam", "churn"):
        return _prepare_pages(c, g)
    B, T, Hkv, D, P = c["B"], c["T"], c["Hkv"], c["D"], c["page"]
    lens, new = _lens(c, g)
    table, pool = _table(_ceil(lens + new, P), g)
    pages = torch.full((pool, Hkv, P * D * 5 // 4), 255, device="cuda", dtype=torch.uint8)  # stale: params are NaN
    dt = TYPES[c["type"]]
    spread = torch.exp(0.5 * torch.randn(Hkv, 1, D, device="cuda", generator=g))  # some channels are larger
    # the rows already cached: keys (rotated, with larger channels) and values, quantised; stale rows behind them
    row, slot = (table >= 0).nonzero(as_tuple=True)
    ids, left = table[row, slot].long(), (lens[row].long() - slot * P).clamp(0, P)
    step = max(1, (1 << 27) // (Hkv * P * D))
    for i in range(0, ids.numel(), step):
        n = ids[i:i + step].numel()
        k = torch.randn(n, Hkv, P, D, device="cuda", generator=g) * spread
        v = torch.randn(n, Hkv, P, D, device="cuda", generator=g)
        parts = []
        for x in (k, v):
            code, s, z = _quantise(x)
            stale = (torch.arange(P, device="cuda") >= left[i:i + step, None])[:, None, :, None]
            parts += [code.reshape(n, Hkv, P // 16, 16, D), s.masked_fill(stale, math.nan).reshape(n, Hkv, P // 16, 16, -1),
                      z.masked_fill(stale, math.nan).reshape(n, Hkv, P // 16, 16, -1)]
        pages[ids[i:i + step]] = _pack(*parts).reshape(n, Hkv, -1)
    st = dict(case=c, pages=pages, table=table, lens=lens, new=new)
    st["k"] = (torch.randn(B, T, Hkv, D, device="cuda", generator=g) * spread[:, 0]).to(dt)
    st["v"] = torch.randn(B, T, Hkv, D, device="cuda", generator=g).to(dt)
    st["kw"] = st["qw"] = None
    if c["norm"]:
        st["kw"] = 0.3 * torch.randn(D, device="cuda", generator=g)
        st["qw"] = 0.3 * torch.randn(D, device="cuda", generator=g)
    st["k_held"], st["v_held"] = torch.empty_like(st["k"]), torch.empty_like(st["v"])
    if c["op"] == "decode":
        st["q"] = torch.randn(B, T, c["Hq"], D, device="cuda", generator=g).to(dt)
        st["o"] = torch.empty_like(st["q"])
    return st


def _prepare_pages(c, g):
    B, P = c["B"], c["page"]
    lens = torch.randint(c["lo"], c["hi"] + 1, (B,), device="cuda", dtype=torch.int32, generator=g)
    row = torch.arange(B, device="cuda", dtype=torch.int32)
    if c["op"] == "beam":  # the beams of a prompt have one length
        base = row // c["beams"] * c["beams"]
        lens = lens[base].contiguous()
    used = _ceil(lens + c["T"], P)
    table, pool = _table(used, g, 0.3)
    # a server's table and pool have one size whatever the requests: room for the longest of them
    wide = _ceil(c["hi"] + c["T"], P)
    table = torch.nn.functional.pad(table, (0, wide - table.shape[1]), value=-1).contiguous()
    pool = (B + c.get("leave", 0)) * wide + int(0.3 * B * wide) + 4
    st = dict(case=c, lens=lens, new=torch.full((B,), c["T"], device="cuda", dtype=torch.int32))
    if c["op"] == "beam":
        # a parent within the beam's own group; the rows of a group share all full pages
        st["parents"] = (base + torch.randint(0, c["beams"], (B,), device="cuda", generator=g)).int()
        shared = torch.arange(wide, device="cuda") < (lens // P)[:, None]
        table = torch.where(shared, table[base], table).contiguous()
    if c["op"] == "churn":
        # rows move up by `leave`; the last ones are admitted empty and get their pages
        fresh = row + c["leave"] >= B
        st["parents"] = torch.where(fresh, -1, row + c["leave"]).int()
        st["new"] = torch.where(fresh, lens, 0).int()
        st["lens"] = torch.where(fresh, 0, lens).int()  # what a row holds before it is written
    refs = torch.zeros(pool, device="cuda", dtype=torch.int32)
    ids = table[table >= 0].long()
    refs.index_add_(0, ids, torch.ones_like(ids, dtype=torch.int32))
    st.update(table=table, refs=refs, counts=torch.zeros(2, device="cuda", dtype=torch.int32))
    size = (c["layers"], pool, c["Hkv"], P * c["D"] * 5 // 4)
    st["pages"] = torch.randint(0, 256, size, device="cuda", dtype=torch.uint8, generator=g)
    return st


_kept = []


def _context():
    """The handle that a user's program keeps."""
    import os
    import sys
    at = os.path.join(os.getcwd(), "win-directml-java_b200")  # the package's parent folder
    if at not in sys.path:
        sys.path.insert(0, at)
    import b200attn
    if not _kept:
        _kept.append(b200attn.Context(0))
    return _kept[0]


# ------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return _own_pages(state) if op in ("draft", "beam", "churn") else _own_cache(state)
    return _plain_pages(state) if op in ("draft", "beam", "churn") else _plain_cache(state)


def _own_cache(st):
    ctx = _context()
    import b200attn
    c = st["case"]
    rope = {"none": b200attn.ROPE_NONE, "neox": b200attn.ROPE_NEOX, "gemma": b200attn.ROPE_GEMMA}[c["rope"]]
    more = dict(new_lens=st["new"], rope_mode=rope, rope_theta=c["theta"], k_norm_w=st["kw"], norm_eps=EPS,
                k_held=st["k_held"], v_held=st["v_held"])
    if c["op"] == "append":
        b200attn.kv4_append(ctx, st["k"], st["v"], st["pages"], st["table"], st["lens"], **more)
        return {"k_held": st["k_held"], "v_held": st["v_held"]}
    b200attn.kv4_decode(ctx, st["q"], st["k"], st["v"], st["pages"], st["table"], st["lens"], st["o"],
                        1.0 / math.sqrt(c["D"]), window=c["window"], q_norm_w=st["qw"], **more)
    return {"o": st["o"], "k_held": st["k_held"], "v_held": st["v_held"]}


def _own_pages(st):
    ctx = _context()
    import b200attn
    c = st["case"]
    if c["op"] == "draft":
        b200attn.pages_free(ctx, st["table"], st["refs"], None, st["lens"], c["page"])
    else:
        b200attn.pages_fork(ctx, st["table"], st["refs"], st["parents"])
    if c["op"] == "churn":
        b200attn.pages_compact(ctx, st["table"], st["refs"], st["pages"], st["counts"])
    b200attn.pages_reserve(ctx, st["table"], st["refs"], st["lens"], st["new"], st["pages"], c["page"], st["counts"])
    return _page_state(st)


# ------------------------------------------------------------------ plain forms of the cache's operators
def _norm_rope(x, w, pos, c):
    """Rows x [B,T,H,D] in 32 bits: zero-centred RMS norm where w is given, then rotation at pos [B,T]."""
    D = x.shape[-1]
    x = x.float()
    if w is not None:
        ss = x.double().square().sum(-1, keepdim=True)
        x = ((x * (ss / D + EPS).sqrt().reciprocal().float()).double() * (1.0 + w.double())).float()
    if c["rope"] == "none":
        return x
    i = torch.arange(D // 2, device=x.device, dtype=torch.float64)
    angle = pos.double()[:, :, None, None] * (1.0 / torch.pow(torch.tensor(c["theta"], dtype=torch.float64), 2.0 * i.cpu() / D)).to(x.device)
    cos, sin = angle.cos(), angle.sin()
    a, b = x[..., :D // 2], x[..., D // 2:]
    if c["rope"] == "gemma":
        a, b = a.double(), b.double()
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).float()
    cos, sin = cos.float(), sin.float()
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _new_rows(st):
    """The new rows as the cache holds them, in 32 bits (absent ones zero), positions and presence [B,T]."""
    c = st["case"]
    t = torch.arange(c["T"], device="cuda")
    pos = st["lens"].long()[:, None] + t
    there = t < st["new"][:, None]
    k = _held(*_quantise(_norm_rope(st["k"], st["kw"], pos, c)))
    v = _held(*_quantise(st["v"].float()))
    return k.masked_fill(~there[..., None, None], 0.0), v.masked_fill(~there[..., None, None], 0.0), pos, there


def _plain_cache(st):
    c = st["case"]
    dt = TYPES[c["type"]]
    k, v, pos, there = _new_rows(st)
    out = {"k_held": k.to(dt), "v_held": v.to(dt)}
    if c["op"] == "append":
        return out
    B, T, Hq, Hkv, D, P = c["B"], c["T"], c["Hq"], c["Hkv"], c["D"], c["page"]
    # every sequence's rows side by side, padded to the longest; what lies behind a context is not looked at
    blocks = st["pages"][st["table"].clamp(min=0).long()]  # [B, max_pages, Hkv, bytes]
    kc, vc = _unpack(blocks.reshape(B, -1, Hkv, P // 16, 20 * D), D)
    del blocks
    cached = torch.arange(kc.shape[1] * P, device="cuda") < st["lens"][:, None]
    kc = kc.transpose(1, 2).reshape(B, Hkv, -1, D).masked_fill_(~cached[:, None, :, None], 0.0)
    vc = vc.transpose(1, 2).reshape(B, Hkv, -1, D).masked_fill_(~cached[:, None, :, None], 0.0)
    q = _norm_rope(st["q"], st["qw"], pos, c).reshape(B, T, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4)
    q = q.reshape(B, Hkv, -1, D)
    n = kc.shape[2]
    s = torch.cat([q @ kc.transpose(-1, -2), q @ k.permute(0, 2, 3, 1)], -1) * (1.0 / math.sqrt(D))
    at = torch.arange(n, device="cuda")
    seen = cached[:, None, :] & (at > pos[..., None] - (c["window"] or 1 << 30))  # [B,T,n]
    t = torch.arange(T, device="cuda")
    fresh = (t <= t[:, None]) & (t > t[:, None] - (c["window"] or 1 << 30))
    seen = torch.cat([seen, (fresh & there[:, None, :]).expand(B, T, T)], -1) & there[..., None]
    s = s.reshape(B, Hkv, -1, T, n + T).masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = (s - torch.where(top == -math.inf, 0.0, top)).exp_()
    p = (p / p.sum(-1, keepdim=True).clamp(min=1e-30)).reshape(B, Hkv, -1, n + T)
    o = p[..., :n] @ vc + p[..., n:] @ v.permute(0, 2, 1, 3)
    o = o.reshape(B, Hkv, Hq // Hkv, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D)
    return {"o": o.to(dt), **out}


# ------------------------------------------------------------------ plain forms of the page operators
def _plain_free(table, refs, keep_from, keep_to, page):
    """Slots that hold no position of [keep_from, keep_to) give their page back."""
    start = torch.arange(table.shape[1], device="cuda") * page
    keep = start < keep_to[:, None]
    if keep_from is not None:
        keep &= start + page > keep_from[:, None]
    gone = (table >= 0) & ~keep
    ids = torch.where(gone, table, 0).long().reshape(-1)
    refs.index_add_(0, ids, -gone.int().reshape(-1))
    table.masked_fill_(gone, -1)


def _plain_fork(table, refs, parents):
    """Row i becomes what row parents[i] was before the call; -1: an empty row."""
    after = torch.where(parents[:, None] >= 0, table[parents.clamp(min=0).long()], -1)
    for_new, for_old = after.clamp(min=0).long().reshape(-1), table.clamp(min=0).long().reshape(-1)
    refs.index_add_(0, for_new, (after >= 0).int().reshape(-1))
    refs.index_add_(0, for_old, -(table >= 0).int().reshape(-1))
    table.copy_(after)


def _plain_compact(table, refs, pages, counts):
    """n live pages: those at n or above move, in order, into the free places below n, in order."""
    live = refs > 0
    n = live.sum()
    at = torch.arange(refs.numel(), device="cuda")
    source = (live & (at >= n)).nonzero()[:, 0]
    target = (~live & (at < n)).nonzero()[:, 0]
    pages[:, target] = pages[:, source]
    refs[target] = refs[source]
    refs[source] = 0
    to = at.int()
    to[source] = target.int()
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], -1))
    counts.copy_(torch.stack([n, torch.tensor(source.numel(), device="cuda")]))


def _plain_reserve(table, refs, lens, new, pages, page, counts):
    """Every slot that positions [lens, lens + new) fall into gets a page of its own: an empty slot a new one, a
    slot whose page other rows hold too (its count at the call's start is above 1) a copy.  New pages are the
    lowest free ones (count 0 at the call's start), given out in the order of rows, then slots.  Where too few are
    free nothing changes.  counts: pages given out, pages missing."""
    start = torch.arange(table.shape[1], device="cuda") * page
    written = (start < (lens + new)[:, None]) & (start + page > lens[:, None]) & (new > 0)[:, None]
    shared = written & (table >= 0) & (refs[table.clamp(min=0).long()] > 1)
    want = (written & (table < 0)) | shared
    free = (refs == 0).nonzero()[:, 0]
    row, slot = want.nonzero(as_tuple=True)
    need = row.numel()
    if need > free.numel():
        counts.copy_(torch.tensor([0, need - free.numel()]))
        return
    got = free[:need]
    copied = shared[row, slot]
    old = table[row, slot].long()[copied]
    pages[:, got[copied]] = pages[:, old]
    refs.index_add_(0, old, torch.full_like(old, -1, dtype=torch.int32))
    refs[got] = 1
    table[row, slot] = got.int()
    counts.copy_(torch.tensor([need, 0]))


def _plain_pages(st):
    c = st["case"]
    if c["op"] == "draft":
        _plain_free(st["table"], st["refs"], None, st["lens"], c["page"])
    else:
        _plain_fork(st["table"], st["refs"], st["parents"])
    if c["op"] == "churn":
        _plain_compact(st["table"], st["refs"], st["pages"], st["counts"])
    _plain_reserve(st["table"], st["refs"], st["lens"], st["new"], st["pages"], c["page"], st["counts"])
    return _page_state(st)


def _page_state(st):
    """What the calls leave; the pages themselves where any is copied."""
    names = ["table", "refs", "counts"] + ([] if st["case"]["op"] == "draft" else ["pages"])
    return {k: st[k] for k in names}


# ------------------------------------------------------------------ the least work
def work(case):
    c = case
    mean = (c["lo"] + c["hi"]) / 2
    new = c["T"] * (0.5 if c.get("ragged") else 1.0)
    if c["op"] in ("decode", "append"):
        rows = c["B"] * new * c["Hkv"] * c["D"]
        nbytes = rows * 2 * (2 + 2) + rows * 1.25 + 4 * c["B"] * (2 + mean / c["page"])  # rows in, rows as held, codes
        if c["op"] == "append":
            return {"bytes": nbytes, "flops": 12.0 * rows}
        seen = min(mean, c["window"]) if c["window"] else mean
        reach = min(mean, c["window"] + new) if c["window"] else mean
        nbytes += c["B"] * reach * c["Hkv"] * 1.25 * c["D"] * (new > 0) + 4.0 * c["B"] * new * c["Hq"] * c["D"]
        return {"bytes": nbytes, "flops": 4.0 * c["B"] * new * c["Hq"] * c["D"] * (seen + (new + 1) / 2)}
    used = (mean + c["T"] + c["page"] / 2) / c["page"]
    nbytes = 8.0 * c["B"] * used  # the table's entries once, each with its count
    page_bytes = 1.25 * c["page"] * c["Hkv"] * c["D"] * c["layers"]
    # beams: the rows whose parent has another child; churn: as many pages move as left
    copied = {"draft": 0.0, "beam": c["B"] * (1 - (1 - 1 / c.get("beams", 1)) ** (c.get("beams", 1) - 1)), "churn": c.get("leave", 0) * used}[c["op"]]
    return {"bytes": nbytes + 2 * copied * page_bytes, "flops": 0.0}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    """Whole numbers have no 64-bit value of their own: the page operators' results are left out.  The codes of
    new rows are whole numbers decided on 32-bit values (part of the definition); what they stand for, and the
    attention, is computed in 64 bits."""
    c = case
    if c["op"] in ("draft", "beam", "churn"):
        return None
    st = prepare(case, seed)
    B, T, Hkv, D, P = c["B"], c["T"], c["Hkv"], c["D"], c["page"]
    f64 = torch.float64
    dev = st["k"].device
    half = D // 2
    inv = torch.tensor([c["theta"] ** (-2.0 * i / D) for i in range(half)], dtype=f64, device=dev)

    def rows(x, w, b, n, first):  # n rows [n,H,D] of sequence b from position `first`, in 64 bits
        y = x[b, :n].to(f64)
        if w is not None:
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * (1 + w.to(f64))
        if c["rope"] == "none":
            return y
        th = (first + torch.arange(n, device=dev, dtype=f64))[:, None, None] * inv
        lo, hi = y[..., :half].clone(), y[..., half:].clone()
        y[..., :half] = lo * torch.cos(th) - hi * torch.sin(th)
        y[..., half:] = hi * torch.cos(th) + lo * torch.sin(th)
        return y

    def rows32(b, n, first):  # the new keys as the 32-bit rows on which the codes are decided
        y = st["k"][b, :n].float()
        if st["kw"] is not None:
            rms = (1 / torch.sqrt((y.to(f64) ** 2).sum(-1, keepdim=True) / D + EPS)).float()
            y = ((y * rms).to(f64) * (1 + st["kw"].to(f64))).float()
        if c["rope"] == "none":
            return y
        th = (first + torch.arange(n, device=dev, dtype=f64))[:, None, None] * inv
        up = f64 if c["rope"] == "gemma" else torch.float32
        cs, sn, lo, hi = torch.cos(th).to(up), torch.sin(th).to(up), y[..., :half].to(up), y[..., half:].to(up)
        return torch.cat([(lo * cs - hi * sn).float(), (lo * sn + hi * cs).float()], -1)

    def store(y):  # the values that the cache holds for rows y
        y = y.unflatten(-1, (D // 32, 32))
        lo = y.min(-1, keepdim=True).values
        s = ((y.max(-1, keepdim=True).values - lo) * FIFTEENTH).half().float()
        z = lo.half().float()
        code = torch.zeros_like(y)
        m = (s > 0).expand_as(y)
        code[m] = torch.clamp(torch.round(((y - z) * (1 / s))[m]), 0, 15)
        return (code.to(f64) * s.to(f64) + z.to(f64)).flatten(-2)

    # where a block holds the code of (key, d), by arithmetic
    key, d = torch.arange(16, device=dev)[:, None], torch.arange(D, device=dev)[None, :]
    r32 = d % 32
    x, j = r32 // 16, (r32 // 8) % 2
    k_byte = ((d // 32 * 8 + key % 8) * 4 + (r32 % 8) // 2) * 8 + x * 4 + 2 * (d % 2) + key // 8
    v_byte = ((d // 32 * 8 + d % 8) * 4 + (key % 8) // 2) * 8 + x * 4 + 2 * (key % 2) + key // 8
    param = ((key % 8) * 2 + key // 8) * (D // 32) + d // 32

    def read(slab, byte, at):  # slab [pages, Hkv, P/16, 20 D] -> [Hkv, pages * P, D]
        code = (slab[..., at + byte].int() >> (4 * j)) & 15
        pr = slab[..., at + 8 * D:at + 10 * D].contiguous().view(torch.float16).to(f64)
        val = code.to(f64) * pr[..., 2 * param] + pr[..., 2 * param + 1]
        return val.transpose(0, 1).reshape(Hkv, -1, D)

    out = {"k_held": torch.zeros(B, T, Hkv, D, dtype=f64, device=dev), "v_held": torch.zeros(B, T, Hkv, D, dtype=f64, device=dev)}
    if c["op"] == "decode":
        out["o"] = torch.zeros(B, T, c["Hq"], D, dtype=f64, device=dev)
    for b in range(B):
        L, n = int(st["lens"][b]), int(st["new"][b])
        if n == 0:
            continue
        kn, vn = store(rows32(b, n, L)), store(st["v"][b, :n].float())
        out["k_held"][b, :n], out["v_held"][b, :n] = kn, vn
        if c["op"] != "decode":
            continue
        ids = st["table"][b, :(L + P - 1) // P].long()
        slab = st["pages"][ids].reshape(-1, Hkv, P // 16, 20 * D)
        K = torch.cat([read(slab, k_byte, 0)[:, :L], kn.transpose(0, 1)], 1)
        V = torch.cat([read(slab, v_byte, 10 * D)[:, :L], vn.transpose(0, 1)], 1)
        q = rows(st["q"], st["qw"], b, n, L).transpose(0, 1).reshape(Hkv, -1, n, D)
        pos = L + torch.arange(n, device=dev)[:, None]
        at = torch.arange(L + n, device=dev)[None, :]
        hide = (at > pos) | ((at <= pos - c["window"]) if c["window"] else torch.zeros_like(at > pos))
        s = torch.einsum("hgnd,hmd->hgnm", q, K) / math.sqrt(D)
        w = torch.softmax(s.masked_fill(hide, -math.inf), -1)
        out["o"][b, :n] = torch.einsum("hgnm,hmd->nhgd", w, V).reshape(n, -1, D)
    return out
