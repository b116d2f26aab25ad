"""A plain numpy model of the paged 4-bit KV cache (include/b200attn.h) in 64 bits, with the code
decisions on 32-bit values as the definition has them.  A cache is held densely: codes and params per
page, kv head, position; `pack` / `unpack` convert to and from the library's bytes by the header's
place formulas."""
import numpy as np

GROUP = 32


def places(D):
    """Byte and nibble shift of every (key, d) of a block's K and V codes, and the params' index."""
    key, d = np.meshgrid(np.arange(16), np.arange(D), indexing="ij")
    y, x = d // 32, d // 16 % 2
    kb = ((y * 8 + key % 8) * 4 + d % 8 // 2) * 8 + x * 4 + 2 * (d % 2) + key // 8
    vb = ((y * 8 + d % 8) * 4 + key % 8 // 2) * 8 + x * 4 + 2 * (key % 2) + key // 8
    shift = 4 * (d // 8 % 2)
    param = ((np.arange(16)[:, None] % 8) * 2 + np.arange(16)[:, None] // 8) * (D // 32) + np.arange(D // 32)
    return kb, vb, shift, param


def pack(kc, ks, vc, vs):
    """codes [..., P, D] uint8, params [..., P, D/32, 2] float16 -> bytes [..., P * D * 5 / 4]."""
    *head, P, D = kc.shape
    kb, vb, shift, param = places(D)
    out = np.zeros((*head, P // 16, 20 * D), np.uint8)
    for byte, at, code, sz in ((kb, 0, kc, ks), (vb, 10 * D, vc, vs)):
        c = code.reshape(*head, P // 16, 16, D)
        for s in (0, 4):
            m = shift == s
            out[..., at + byte[m]] |= (c[..., m] << s).astype(np.uint8)
        w = np.zeros((*head, P // 16, 16 * (D // 32), 2), np.float16)
        w[..., param.reshape(-1), :] = sz.reshape(*head, P // 16, 16 * (D // 32), 2)
        out[..., at + 8 * D:at + 10 * D] = w.view(np.uint8).reshape(*head, P // 16, 2 * D)
    return out.reshape(*head, P * D * 5 // 4)


def unpack(raw, D):
    """bytes [..., P * D * 5 / 4] -> kc, ks, vc, vs as `pack` takes them."""
    *head, n = raw.shape
    P = n * 4 // (5 * D)
    kb, vb, shift, param = places(D)
    blk = np.ascontiguousarray(raw).reshape(*head, P // 16, 20 * D)
    got = []
    for byte, at in ((kb, 0), (vb, 10 * D)):
        got.append(((blk[..., at + byte] >> shift) & 15).reshape(*head, P, D))
        w = np.ascontiguousarray(blk[..., at + 8 * D:at + 10 * D]).view(np.float16).reshape(*head, P // 16, -1, 2)
        got.append(w[..., param.reshape(-1), :].reshape(*head, P, D // 32, 2))
    return got


def quantise(x):
    """Rows [..., D] (32-bit) -> codes uint8, params float16 [..., D/32, 2]."""
    g = np.ascontiguousarray(x, np.float32).reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    with np.errstate(all="ignore"):
        lo, hi = g.min(-1), g.max(-1)
        s = ((hi - lo) * np.float32(1.0 / 15.0)).astype(np.float16)
        z = lo.astype(np.float16)
        sf, zf = s.astype(np.float32), z.astype(np.float32)
        inv = np.where(sf > 0, np.float32(1) / sf, np.float32(0))
        c = np.clip(np.rint((g - zf[..., None]) * inv[..., None]), 0, 15)
    bad = ~(np.isfinite(g).all(-1) & np.isfinite(sf) & np.isfinite(zf))
    c = np.where(bad[..., None], 0, c).astype(np.uint8)
    sz = np.stack([s, z], -1)
    sz[bad] = np.nan
    return c.reshape(x.shape), sz


def values(code, sz):
    """What codes [..., D] with params [..., D/32, 2] stand for, in 64 bits."""
    g = code.reshape(*code.shape[:-1], code.shape[-1] // GROUP, GROUP).astype(np.float64)
    return (g * sz[..., 0:1].astype(np.float64) + sz[..., 1:2].astype(np.float64)).reshape(code.shape)


def norm_rope(x, w, pos, mode, theta, eps=np.float32(1e-6), bits=32):
    """Rows x [T,H,D] at positions pos [T].  bits 32: the rounding steps of the definition (what the
    codes are decided on); 64: plain."""
    D = x.shape[-1]
    x = x.astype(np.float32)
    if bits == 64:
        x = x.astype(np.float64)
    if w is not None:
        ss = (x.astype(np.float64) ** 2).sum(-1, keepdims=True)
        rms = 1.0 / np.sqrt(ss / D + float(eps))
        if bits == 32:
            x = ((x * rms.astype(np.float32)).astype(np.float64) * (1.0 + w.astype(np.float64))).astype(np.float32)
        else:
            x = x * rms * (1.0 + w.astype(np.float64))
    if mode is None:
        return x
    i = np.arange(D // 2)
    a = np.asarray(pos, np.float64)[:, None, None] * (1.0 / theta ** (2.0 * i / D))
    c, s = np.cos(a), np.sin(a)
    lo, hi = x[..., :D // 2], x[..., D // 2:]
    if bits == 32 and mode == "neox":
        c, s = c.astype(np.float32), s.astype(np.float32)
    elif bits == 32:
        lo, hi = lo.astype(np.float64), hi.astype(np.float64)
    y = np.concatenate([lo * c - hi * s, lo * s + hi * c], -1)
    return y.astype(np.float32) if bits == 32 else y


def attend(q, K, V, pos, window, scale):
    """q [T,Hq,D] (64-bit, rotated), K, V [n,Hkv,D] (keys 0..n-1), query t at pos[t] -> [T,Hq,D]."""
    T, Hq, D = q.shape
    Hkv = K.shape[1]
    G = Hq // Hkv
    at = np.arange(K.shape[0])[None, :]
    see = at <= pos[:, None]
    if window:
        see &= at > pos[:, None] - window
    out = np.zeros((T, Hq, D))
    for h in range(Hq):
        s = (q[:, h] @ K[:, h // G].T) * scale
        s = np.where(see, s, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        out[:, h] = (p @ V[:, h // G]) / p.sum(-1, keepdims=True)
    return out
