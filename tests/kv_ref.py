"""Plain 64-bit forms of the key/value cache's operators (comp_amd.kv), for its tests."""

import numpy as np

from oracle import oracle as O


def kept(x, fmt):
    """f32 [T][H][D] -> f64 [T][H][D]: what a cache of this format keeps of x, by the oracle's ggml quantizers."""
    t, h, d = x.shape
    if t == 0:
        return np.zeros(x.shape)
    rows = np.ascontiguousarray(x, dtype=np.float32).reshape(t * h, d)
    if fmt == "q8_0":
        q, s, _ = O.quantize("q8_0", rows)
        return (q.astype(np.float64).reshape(t * h, -1, 32) * s.astype(np.float64)[:, :, None]).reshape(t, h, d)
    blocks = np.frombuffer(O.quantize_q4_0_weights(rows), np.uint8).reshape(t * h, d // 32, 18)
    s = blocks[:, :, :2].copy().view(np.float16).astype(np.float64)
    q = np.concatenate([blocks[:, :, 2:] & 15, blocks[:, :, 2:] >> 4], axis=2).astype(np.float64) - 8
    return (q * s).reshape(t, h, d)


def attend(q, keys, values, counts, *, scale=None, softcap=0.0, window=0, prefix=None, slopes=None):
    """q [T][heads][D], keys / values: a list of [n][kv heads][D] a sequence, counts: query rows a sequence ->
    (out [T][heads][D], lse [T][heads]) in f64, by the definition."""
    q = np.asarray(q, np.float64)
    t, heads, d = q.shape
    scale = d**-0.5 if scale is None else scale
    out, lse = np.zeros(q.shape), np.full((t, heads), -np.inf)
    first = 0
    for s, (k, v, n) in enumerate(zip(keys, values, counts)):
        length, j = k.shape[0], np.arange(k.shape[0])
        i = np.arange(length - n, length)[:, None]
        seen = j <= i
        if prefix is not None:
            seen = seen | (j < prefix[s])
        if window:
            seen = seen & (i - j < window)
        for h in range(heads):
            kv = h // (heads // k.shape[1])
            with np.errstate(invalid="ignore", over="ignore"):
                x = scale * (q[first : first + n, h] @ k[:, kv].T)
            if softcap:
                x = softcap * np.tanh(x / softcap)
            if slopes is not None:
                x = x - float(slopes[h]) * np.abs(i - j)
            x = np.where(seen, x, -np.inf)
            if not x.size:
                continue
            top = x.max(axis=1, keepdims=True)
            top[top == -np.inf] = 0
            p = np.exp(x - top)
            total = p.sum(axis=1)
            some = total > 0
            out[first : first + n, h][some] = (p @ v[:, kv])[some] / total[some, None]
            lse[first : first + n, h][some] = top[some, 0] + np.log(total[some])
        first += n
    return out, lse
