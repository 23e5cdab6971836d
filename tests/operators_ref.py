"""Plain 64-bit implementations of the operators that include/zrnn.h declares under "Operators of a decoding step"."""
import math

import numpy as np
import torch

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# a rounding to the type is off by at most half a step, relative to the value
HALF_STEP = {k: torch.finfo(t).eps / 2 for k, t in TYPES.items()}


def pack(x, heads, d):
    """x [S, B, heads * d] float64 NumPy -> (codes [B, S, heads, G * 16] uint8, scales [B, S, heads, G] float16)."""
    S, B = x.shape[:2]
    G = -(-d // 32)
    g = np.zeros((B, S, heads, G * 32))
    g[..., :d] = np.asarray(x).reshape(S, B, heads, d).transpose(1, 0, 2, 3)
    g = g.reshape(B, S, heads, G, 32)
    with np.errstate(all="ignore"):
        a = np.abs(g).max(-1)
        s = np.minimum(a.astype(np.float32) * np.float32(1.0 / 7.0), np.float32(9352.0)).astype(np.float16)
        s = np.where(np.isfinite(a), s, np.float16(np.nan))
        ok = (s > 0)[..., None]
        q = np.where(ok, np.clip(np.rint(g / np.where(ok, s[..., None].astype(np.float64), 1.0)), -7, 7), 0)
    u = (np.nan_to_num(q) + 8).astype(np.uint8).reshape(B, S, heads, G * 32)
    return u[..., 0::2] | (u[..., 1::2] << 4), s


def unpack(codes, scales, d):
    """[B, S, heads, d] float64: q * s rounded to half precision."""
    u = np.empty(codes.shape[:-1] + (codes.shape[-1] * 2,))
    u[..., 0::2], u[..., 1::2] = codes & 15, codes >> 4
    v = (u - 8) * np.repeat(scales.astype(np.float64), 32, -1)
    with np.errstate(all="ignore"):
        return v.astype(np.float16).astype(np.float64)[..., :d]


def attend(v, q, lens, offsets, scale, mask=None):
    """v [B, S, heads, d], q [N, heads * d] float64 -> ([N, heads, d], the largest sum of |scale q v| over d per column and head)."""
    B, S, heads, d = v.shape
    N = q.shape[0]
    cols = N // B
    out, mag = np.zeros((N, heads, d)), np.zeros((N, heads))
    for c in range(N):
        b = c // cols
        lo, hi = max(int(offsets[b]), 0), min(int(offsets[b]) + int(lens[b]), S)
        if hi <= lo or (mask is not None and mask[c] == 0):
            continue
        w, qc = v[b, lo:hi], q[c].reshape(heads, d)
        z = np.einsum("hd,shd->hs", qc, w) * scale
        p = np.exp(z - z.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        out[c] = np.einsum("hs,shd->hd", p, w)
        mag[c] = (np.einsum("hd,shd->hs", np.abs(qc), np.abs(w)) * abs(scale)).max(1)
    return out, mag


def act(x, name):
    if name == "tanh":
        return torch.tanh(x)
    if name == "sigmoid":
        return torch.sigmoid(x)
    if name == "relu":
        return torch.where(torch.isnan(x), x, torch.clamp(x, min=0))
    if name == "gelu":
        return 0.5 * x * (1 + torch.erf(x / math.sqrt(2)))
    if name == "silu":
        return x * torch.sigmoid(x)
    return x


def select(z, scores, beam, k, lse=None, done=None, eos=1):
    """float32 NumPy arrays; the candidates' values are float32 by definition.  Returns (values, words, parents)."""
    rows, V = z.shape
    n = rows // beam
    val, word, parent = np.full((n, k), -np.inf, np.float32), np.full((n, k), -1, np.int32), np.full((n, k), -1, np.int32)
    with np.errstate(all="ignore"):
        c = z.astype(np.float32)
        if lse is not None:
            c = (c - lse[:, None].astype(np.float32)).astype(np.float32)
        c = (scores[:, None].astype(np.float32) + c).astype(np.float32)
    if done is not None:
        over = done != 0
        c[over] = -np.inf
        c[over, eos] = scores[over]
    c = np.where(np.isnan(c), np.float32(-np.inf), c).reshape(n, beam * V)
    for b in range(n):
        at = np.argsort(-c[b], kind="stable")[:k]
        at = at[c[b][at] > -np.inf]
        val[b, :len(at)], word[b, :len(at)], parent[b, :len(at)] = c[b][at], at % V, at // V + b * beam
    return val, word, parent


def reorder(x, parents, n):
    out = np.zeros((n,) + x.shape[1:], x.dtype)
    ok = parents >= 0
    out[ok] = x[parents[ok]]
    return out
