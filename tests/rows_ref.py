"""The rows operators (include/speech_hip.h, speech_rows_*) stated in numpy, 64 bits, for the tests."""
import numpy as np

BLOCK = 128


def mix64(z):
    with np.errstate(over="ignore"):
        z = np.asarray(z, np.uint64) + np.uint64(0x9E3779B97F4A7C15)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        return z ^ (z >> np.uint64(31))


def kept(p, seed, keys, cols):
    """the mask of dropout: rows of len(keys), bool"""
    keys = np.asarray(keys).astype(np.uint64)
    with np.errstate(over="ignore"):
        fk = mix64(mix64(np.uint64((seed & (2 ** 64 - 1)) ^ 0xD1B54A32D192ED03)) ^ keys)
        h = (fk & np.uint64(0xFFFFFFFF)).astype(np.uint32)[:, None] ^ (np.arange(cols, dtype=np.uint32) * np.uint32(0x9E3779B9))[None, :]
        h = (h ^ (h >> np.uint32(16))) * np.uint32(0x85EBCA6B)
        h = (h ^ (h >> np.uint32(13))) * np.uint32(0xC2B2AE35)
        h = (h ^ (h >> np.uint32(16))) + (fk >> np.uint64(32)).astype(np.uint32)[:, None]
    return h >= np.uint32(int(np.floor(p * 2.0 ** 32)))


def dropped(x, p, mask):
    return x if p == 0.0 else np.where(mask, x / (1.0 - p), 0.0)


def e4m3_values():
    """what each of the 256 bytes stands for"""
    b = np.arange(256)
    s, e, m = np.where(b & 128, -1.0, 1.0), (b >> 3) & 15, b & 7
    v = s * np.where(e == 0, m * 2.0 ** -9, (1.0 + m / 8.0) * 2.0 ** (e.astype(np.float64) - 7))
    v[(b & 127) == 127] = np.nan
    return v


def to_e4m3(v):
    """bytes of v (at most 448 in magnitude, or no finite number: NaN), nearest even"""
    table = e4m3_values()[:127]
    a = np.abs(v)
    bad = ~np.isfinite(v)
    a = np.where(bad, 0.0, a)
    hi = np.clip(np.searchsorted(table, a, side="left"), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = table[hi] - a, a - table[lo]
    pick = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    out = np.where(np.signbit(v), pick | 128, pick).astype(np.uint8)
    return np.where(bad, np.uint8(127), out)


def exponents(v):
    """biased exponent of each block of 128 columns: the smallest e in 0 ... 254 with max |v| 2^(127 - e) <= 448, over finite values"""
    rows, cols = v.shape
    nb = -(-cols // BLOCK)
    a = np.zeros((rows, nb * BLOCK))
    a[:, :cols] = np.where(np.isfinite(v), np.abs(v), 0.0)
    amax = a.reshape(rows, nb, BLOCK).max(2)
    m, e = np.frexp(amax)                                      # amax = m 2^e, 0.5 <= m < 1; 448 = 0.875 2^9
    e = np.where(m > 0.875, e - 8, e - 9) + 127
    return np.where(amax == 0.0, 0, np.maximum(e, 0)).astype(np.uint8)


def spread(e, cols):
    """the scale of each column"""
    return np.repeat(2.0 ** (e.astype(np.float64) - 127), BLOCK, axis=1)[:, :cols]


def quantized(v):
    e = exponents(v)
    return to_e4m3(v / spread(e, v.shape[1])), e


def stands_for(q, e):
    return e4m3_values()[q] * spread(e, q.shape[1])
