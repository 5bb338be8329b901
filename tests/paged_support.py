"""Caller-owned paged caches for the row, attention and logits operators, and
their plain implementations in 64 bits on the CPU."""
import numpy as np
import torch

from attention_support import BLOCK, K_BYTE, K_OFF, KS_OFF, PAGE_POS, S_SLOT, V_BYTE, V_OFF, VS_OFF

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# half a step of each type, relative to the value
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


class Cache:
    """Slots of random codes and scales over pages in random order.  Bytes no
    slot uses, behind each slot's length included, hold garbage: codes of any
    value and scales of NaN, infinity and the largest finite value."""

    def __init__(self, seed, lengths, kv_heads, layers=2, layer=1, spare_pages=2, spare_columns=1, peak=1.0):
        rng = self.rng = np.random.default_rng(seed)
        self.kv_heads, self.layers, self.layer, self.lengths = kv_heads, layers, layer, list(lengths)
        need = [(n + PAGE_POS - 1) // PAGE_POS for n in lengths]
        self.max_pages = max(1, max(need, default=0)) + spare_columns
        self.num_pages = sum(need) + spare_pages
        self.page_bytes = layers * kv_heads * BLOCK
        order = rng.permutation(self.num_pages)
        self.table = np.full((len(need), self.max_pages), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        pool = rng.integers(0, 256, (self.num_pages, layers, kv_heads, BLOCK), dtype=np.uint8)
        junk = np.array([np.nan, np.inf, -np.inf, np.finfo(np.float32).max], np.float32)
        pool[..., KS_OFF:V_OFF] = rng.choice(junk, pool.shape[:3] + (128,)).view(np.uint8)
        self.k = [rng.integers(-127, 128, (n, kv_heads, 64)).astype(np.int8) for n in lengths]
        self.v = [rng.integers(-127, 128, (n, kv_heads, 64)).astype(np.int8) for n in lengths]
        self.ks = [(peak * rng.uniform(0.004, 0.02, (n, kv_heads))).astype(np.float32) for n in lengths]
        self.vs = [(2.0 ** rng.uniform(-9, -3, (n, kv_heads))).astype(np.float32) for n in lengths]
        self.pool = pool
        for s, n in enumerate(lengths):
            for i in range(need[s]):
                lo, hi = i * PAGE_POS, min(n, (i + 1) * PAGE_POS)
                for h in range(kv_heads):
                    rec = pool[self.table[s, i], layer, h]
                    c = hi - lo
                    rec[K_OFF + K_BYTE[:c]] = self.k[s][lo:hi, h].view(np.uint8)
                    rec[V_OFF + V_BYTE[:c]] = self.v[s][lo:hi, h].view(np.uint8)
                    rec[KS_OFF:KS_OFF + 256].view(np.float32)[S_SLOT[:c]] = self.ks[s][lo:hi, h]
                    rec[VS_OFF:VS_OFF + 256].view(np.float32)[:c] = self.vs[s][lo:hi, h]

    def keys(self, s):
        return self.k[s].astype(np.float64) * self.ks[s][..., None]

    def values(self, s):
        return self.v[s].astype(np.float64) * self.vs[s][..., None]

    def device(self, cuda):
        """(page_table, pool, page_bytes, layer) on the device."""
        return (torch.from_numpy(self.table).to(cuda), torch.from_numpy(self.pool.reshape(-1)).to(cuda),
                self.page_bytes, self.layer)


def records(pool, cache):
    """Codes and scales [pages, kv heads, 64 positions, ...] of a pool's bytes in the cache's layer."""
    rec = pool.reshape(cache.num_pages, cache.layers, cache.kv_heads, BLOCK)[:, cache.layer]
    scales = np.ascontiguousarray(rec[..., KS_OFF:V_OFF]).view(np.float32)
    return (rec[..., K_OFF + K_BYTE].view(np.int8), rec[..., V_OFF + V_BYTE].view(np.int8), scales[..., S_SLOT],
            scales[..., 64:])


def attend(q, keys, values, position, window=0, scale=0.125):
    """(out, size, reach) of one query [heads, 64] at `position` (it sees that
    position and those before) in 64 bits: out [heads, 64], size the same sums
    over |v|, reach [heads] the largest scale * sum |q||k|."""
    heads, kv = q.shape[0], keys.shape[1]
    first = max(0, position + 1 - window) if window else 0
    k, v = keys[first:position + 1], values[first:position + 1]
    out, size, reach = np.zeros((heads, 64)), np.zeros((heads, 64)), np.zeros(heads)
    if position < 0:
        return out, size, reach
    for h in range(heads):
        g = h // (heads // kv)
        s = scale * (k[:, g] @ q[h])
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h], size[h] = p @ v[:, g], p @ np.abs(v[:, g])
        reach[h] = scale * (np.abs(k[:, g]) @ np.abs(q[h])).max()
    return out, size, reach


def bound(kind, out, size, reach, count, largest):
    """How far an attention output may be from the 64-bit one, by arithmetic:
    - a score is a sum of 64 products and two scalings in fp32, off by at most
      (64 + 4) steps of 2^-23 of scale * sum |q||k| (each addition may
      truncate), and a difference of two such scores with the running maximum
      rounds once more: x is off by d <= 72 * 2^-23 * (2 * reach + 1);
    - exp adds 2^-21, a probability rounds by half a step of fp16 (2^-11) for
      16-bit types, for fp32 it is two halves (2^-21); both the sum over v and
      the total carry the factor, the sums themselves round within 2^-18;
    - bf16 callers of the prompt get keys and values as code * scale in fp16:
      a key element is off by two roundings of the product (2 * 2^-11), so a
      score by 2^-10 * reach, a value by its scale's rounding and the
      product's (2 * 2^-11);
    - below fp16's normal range a probability is off by 2^-25 of one that is
      at least 2^-1 (fp32: 2^-36, the second half's);
    - the result rounds by half a step of its type."""
    d = 72 * 2.0 ** -23 * (2 * reach[:, None] + 1)
    p = {"f32": 2.0 ** -21, "f16": 2.0 ** -11, "bf16": 3 * 2.0 ** -11}[kind]
    if kind == "bf16":
        d = d + 2 * 2.0 ** -10 * reach[:, None]
    tiny = (2.0 ** -35 if kind == "f32" else 2.0 ** -24) * count * largest
    return size * (2 * (np.expm1(d) + 2.0 ** -21) + p + 2.0 ** -18) + tiny + HALF_STEP[kind] * (np.abs(out) + 1e-30)


def quantized(x):
    """(codes, scales) of float32 [..., 64] by the definition's fp32 steps."""
    x = x.astype(np.float32)
    peak = np.abs(x).max(-1)
    scale = np.where(peak > 0, peak / np.float32(127), np.float32(1)).astype(np.float32)
    inverse = (np.float32(1) / scale).astype(np.float32)
    codes = np.clip(np.rint(x * inverse[..., None]), -128, 127).astype(np.int8)
    return codes, scale


def processed(x, tokens=None, prompt=0, repetition=None, frequency=None, presence=None, bias=(), mask=None,
              dtype=np.float32):
    """One row of logits by the definition, every step rounded to `dtype`."""
    x = x.astype(dtype).copy()
    n = x.size
    tokens = [] if tokens is None else list(tokens)
    for v in sorted({t for t in tokens if 0 <= t < n}):
        if repetition is not None:
            r = dtype(repetition)
            x[v] = x[v] / r if x[v] > 0 else x[v] * r
        times = tokens[prompt:].count(v)
        if times and frequency is not None:
            x[v] = x[v] - dtype(frequency) * dtype(times)
        if times and presence is not None:
            x[v] = x[v] - dtype(presence)
    for v, b in dict(bias).items():
        if 0 <= v < n:
            x[v] = x[v] + dtype(b)
    if mask is not None:
        for v in range(n):
            if v >= 32 * len(mask) or not (int(mask[v >> 5]) >> (v & 31)) & 1:
                x[v] = -np.inf
    return x
