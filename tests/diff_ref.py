"""64-bit forms of the paged-cache append and of differential attention, and the bounds the tests hold the kernels to."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from espetero_b200 import capi, workloads as wl

U16 = {wl.F16: 2.0 ** -11, wl.BF16: 2.0 ** -8}  # half a step, relative
SUB16 = {wl.F16: 2.0 ** -25, wl.BF16: 0.0}       # half a subnormal step


def rotate64(x, pos, inv_freq, maps, adjacent):
    """x [rows, heads, HD] float64 -> rotated, and |x cos| + |y sin| per element (what the fp32 error is relative to)."""
    rows, heads, HD = x.shape
    D, n = HD // maps, len(inv_freq)
    y = x.reshape(rows, heads, maps, D).copy()
    mag = np.abs(y)
    a = pos.astype(np.float64)[:, None] * inv_freq.astype(np.float64)[None, :]
    c, s = np.cos(a)[:, None, None, :], np.sin(a)[:, None, None, :]
    lo, hi = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if adjacent else (slice(0, n), slice(n, 2 * n))
    u, v = y[..., lo].copy(), y[..., hi].copy()
    y[..., lo], y[..., hi] = u * c - v * s, v * c + u * s
    mag[..., lo] = mag[..., hi] = np.abs(u) + np.abs(v)
    return y.reshape(rows, heads, HD), mag.reshape(rows, heads, HD)


def keys_values(w, i, kvh):
    """Cached and own K, V [P + M, HD] (float64) of tree i for one kv head, and the largest scale of its V pages (1 for 16-bit pools)."""
    t = w.trees[i]
    P, M, base, HD = int(t["P"]), int(t["M"]), int(t["base"]), w.HD
    cols = slice(kvh * HD, (kvh + 1) * HD)
    out, unit = [], 1.0
    pool = w.kv[w.kv_base:].reshape(-1)[:w.n_blocks * 2 * w.bt * w.kv_ld].reshape(w.n_blocks, 2, w.bt, w.kv_ld)
    for which, fresh in ((0, w.Kb), (1, w.Vb)):
        j = np.arange(P)
        b = w.blocks[int(t["table"]) + j // w.bt] if P else np.zeros(0, dtype=np.int64)
        raw = pool[b, which, j % w.bt][:, cols]
        if w.kv_dtype == wl.E4M3:
            kept = wl.e4m3_decode(raw).astype(np.float64) * w.kv_scales[b, which, kvh].astype(np.float64)[:, None]
            if which == 1 and P:
                unit = max(float(w.kv_scales[b, 1, kvh].max()), 1.0 if M else 0.0)
        else:
            kept = wl.from_bits16(raw, w.kv_dtype).astype(np.float64)
        out.append(np.concatenate([kept, wl.from_bits16(fresh[base:base + M, cols], w.q_dtype).astype(np.float64)]))
    return out[0], out[1], unit


def visible(w, i):
    """[M, P + M] truth values."""
    t = w.trees[i]
    P, M, base = int(t["P"]), int(t["M"]), int(t["base"])
    own = np.zeros((M, M), dtype=bool)
    for r in range(M):
        if w.anc_mask is not None:
            own[r] = [(int(w.anc_mask[base + r]) >> j) & 1 for j in range(M)]
        else:
            seg, _, anc, _ = (int(x) for x in w.desc[base + r])
            j = np.arange(M)
            own[r] = (j < anc) | ((j >= seg) & (j <= r))
    return np.concatenate([np.ones((M, P), dtype=bool), own], axis=1)


def diff64(w, lam, norm_w, eps, out_scale, p_unit, rows_of=None):
    """O [rows, H * HD] in float64 and the largest error a right kernel may have, per element.

    lam [rows, H] (or broadcastable). p_unit: half a step of the type the softmax weights are rounded to (0: not rounded).
    The bound: a score of D dims carries (D + 2) 2^-24 sum |q k| scale from its fp32 products and sums, an exponential twice that
    plus 2^-21, a sum of n weights at most n 2^-24, a weight p_unit: relative to A = P_1 |V| + lam P_2 |V| this is e1, and with
    16-bit weights that fall under fp16's normal range half a subnormal step per key more. D's error e then passes the norm:
    |dO| <= f |w| (e + |D| ||e|| / sqrt(||D||^2 + HD eps)), and the result is rounded once."""
    HD, G, d = w.HD, w.G, w.HD // 2
    O = np.zeros((w.n_rows, w.H, HD))
    tol = np.zeros_like(O)
    Q = wl.from_bits16(w.Q, w.q_dtype).astype(np.float64).reshape(w.n_rows, w.H, HD)
    lam = np.broadcast_to(np.asarray(lam, dtype=np.float64), (w.n_rows, w.H))
    wt = np.ones(HD) if norm_w is None else norm_w.astype(np.float64)
    for i, t in enumerate(w.trees):
        base, M = int(t["base"]), int(t["M"])
        if M == 0:
            continue
        vis = visible(w, i)
        n = vis.shape[1]
        for kvh in range(w.Hkv):
            K, V, unit = keys_values(w, i, kvh)
            with np.errstate(invalid="ignore"):
                Vz = np.where(np.isfinite(V), V, 0.0)  # a key nobody sees may hold anything
                Kz = np.where(np.isfinite(K), K, 0.0)
            for h in range(kvh * G, (kvh + 1) * G):
                D, A, sub = np.zeros((M, HD)), np.zeros((M, HD)), np.zeros((M, HD))
                e1 = np.zeros((M, 1))
                for c, sign in ((0, 1.0), (1, -1.0)):
                    q, k = Q[base:base + M, h, c * d:(c + 1) * d], Kz[:, c * d:(c + 1) * d]
                    s = np.where(vis, q @ k.T * w.scale, -np.inf)
                    es = np.where(vis, np.abs(q) @ np.abs(k).T, 0.0).max(axis=1, keepdims=True, initial=0.0) * w.scale * (d + 2) * 2.0 ** -24
                    top = s.max(axis=1, keepdims=True, initial=-np.inf)
                    p = np.exp(s - np.where(np.isfinite(top), top, 0.0))
                    tot = p.sum(axis=1, keepdims=True)
                    p = np.divide(p, tot, out=np.zeros_like(p), where=tot > 0)
                    f = np.ones((M, 1)) if c == 0 else lam[base:base + M, h][:, None]
                    D += sign * f * (p @ Vz)
                    A += np.abs(f) * (p @ np.abs(Vz))
                    if p_unit:
                        # over E4M3 pools the weight carries its page's scale, in units of the largest: a code is at most 448
                        raw = np.where(vis, 1.0, 0.0) @ (np.abs(Vz) if w.kv_dtype != wl.E4M3 else np.full_like(Vz, 448.0 * unit))
                        sub += np.abs(f) * (2.0 ** -25 if p_unit < 2.0 ** -9 else 0.0) * np.divide(raw, tot, out=np.zeros_like(raw), where=tot > 0)
                    e1 = np.maximum(e1, 2 * es + 2.0 ** -21 + (n + 8) * 2.0 ** -24 + p_unit)
                e = e1 * A + sub
                if norm_w is None:
                    fac, grow = np.full((M, 1), out_scale), np.zeros((M, 1))
                else:
                    ms = (D * D).mean(axis=1, keepdims=True)
                    fac = np.where(ms > 0, out_scale / np.sqrt(np.maximum(ms + eps, 1e-300)), 0.0)
                    grow = np.sqrt((e * e).sum(axis=1, keepdims=True)) / np.sqrt(np.maximum((D * D).sum(axis=1, keepdims=True) + HD * eps, 1e-300))
                o = fac * wt * D
                O[base:base + M, h] = o
                tol[base:base + M, h] = 1.02 * np.abs(fac * wt) * (e + np.abs(D) * grow) / np.maximum(1e-3, 1 - grow) + (U16[w.q_dtype] + 2.0 ** -20) * np.abs(o) + SUB16[w.q_dtype] + 1e-30
    return O.reshape(w.n_rows, -1), tol.reshape(w.n_rows, -1)


# ---------------------------------------------------------------------------------------------- host checks without a GPU
_GLUE = """
#include "launch.h"
extern "C" int glue_append(const esp_attn_shape* s, const esp_kv_append_args* a) { return esp::check_kv_append(*s, *a); }
extern "C" int glue_diff(const esp_attn_shape* s, const esp_attn_args* a, const esp_diff_args* d) {
  return esp::check_diff_pass(*s, s->tile_rows, true, *a, *d);
}
extern "C" unsigned long glue_size(int i) { return i ? sizeof(esp_diff_args) : sizeof(esp_kv_append_args); }
"""


@pytest.fixture(scope="session")
def call_checks(tmp_path_factory):
    """The library's own argument checks, which need no context and no device."""
    capi.load()  # the glue's symbols come from it
    at = tmp_path_factory.mktemp("glue")
    src, so = at / "glue.cpp", at / "glue.so"
    src.write_text(_GLUE)
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "espetero_b200", "csrc")
    subprocess.run(["g++", "-std=c++20", "-shared", "-fPIC", "-I", csrc, "-I", "/usr/local/cuda/include", str(src), "-o", str(so), capi.LIB_PATH], check=True)
    lib = ctypes.CDLL(str(so))
    lib.glue_size.restype = ctypes.c_ulong
    assert lib.glue_size(0) == ctypes.sizeof(capi.AppendArgs) and lib.glue_size(1) == ctypes.sizeof(capi.DiffArgs)

    class Checks:
        @staticmethod
        def append(shape, a):
            return lib.glue_append(ctypes.byref(shape), ctypes.byref(a))

        @staticmethod
        def diff(shape, a, d):
            return lib.glue_diff(ctypes.byref(shape), ctypes.byref(a), ctypes.byref(d))

    return Checks
