"""The 4-bit formats and their products in 64 bits, straight from their definitions (numpy, on the host)."""
import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([m / 512 for m in range(8)] + [(8 + m) / 8 * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:-1])
GROUP = {"nvfp4": 16, "mxfp4": 32}


def nearest(x, table):
    """Index of the nearest entry of an ascending table, ties to the even index, beyond the last entry the last."""
    mids = (table[1:] + table[:-1]) / 2
    below, above = np.searchsorted(mids, x, "left"), np.searchsorted(mids, x, "right")
    return np.where(below % 2 == 0, below, above)


def pow2_of_rows(x):
    """x [rows, n] -> the least power of two >= amax / 2688 (finite values), at least 2^-100; 1 for a row of zeros."""
    a = np.where(np.isfinite(x), np.abs(x), 0).max(axis=1, initial=0)
    out = np.ones(len(a))
    for i, v in enumerate(a):
        if v > 0:
            j = -100
            while v > 2688 * 2.0 ** j:
                j += 1
            out[i] = 2.0 ** j
    return out


def quantize_groups(x, gmax, p, fmt):
    """x [..., n] in 64 bits, gmax [...] the largest magnitude of its group (NaN: the group holds a NaN or an infinity), p [...] the
    row's power of two -> (codes [..., n], scale bytes [...])."""
    bad = ~np.isfinite(gmax)
    g = np.where(bad, 0, gmax)
    if fmt == "nvfp4":
        byte = nearest(g / 6 / p, E4M3)
        s = E4M3[byte] * p
        nan = 0x7F
    else:
        with np.errstate(divide="ignore"):
            e = np.where(g > 0, np.frexp(g)[1] - 1 - 2, -127)
        e = np.maximum(e, -127)
        byte, s, nan = e + 127, 2.0 ** e, 0xFF
    dead = bad | (s == 0)
    q = np.where(dead[..., None], 0, x) / np.where(dead, 1, s)[..., None]
    code = nearest(np.abs(q), E2M1)
    return np.where(q < 0, code + 8, code).astype(np.uint8), np.where(bad, nan, byte).astype(np.uint8)


def quantize_dense(x, fmt):
    """x [N, K] -> (codes [N, K], scale bytes [N, groups], powers of two [N] or None)."""
    x = np.asarray(x, np.float64)
    N, K = x.shape
    n = GROUP[fmt]
    full = np.zeros((N, -(-K // n) * n))
    full[:, :K] = x
    p = pow2_of_rows(x) if fmt == "nvfp4" else None
    gr = full.reshape(N, -1, n)
    gmax = np.where(np.isfinite(gr).all(axis=2), np.abs(gr).max(axis=2, initial=0), np.nan)
    codes, s = quantize_groups(gr, gmax, 1.0 if p is None else p[:, None], fmt)
    return codes.reshape(N, -1)[:, :K], s, p


def quantize_blocks(vals, rowptr, colidx, fmt):
    """vals [nnzb, 16, 16] -> (codes [nnzb, 16, 16], scale bytes [nnzb, 16], powers of two [M] or None)."""
    v = np.asarray(vals, np.float64)
    brow = np.repeat(np.arange(len(rowptr) - 1), np.diff(rowptr))
    gmax = np.where(np.isfinite(v).all(axis=2), np.abs(v).max(axis=2), np.nan)
    if fmt == "nvfp4":
        p = np.ones((len(rowptr) - 1, 16))
        for r in range(len(rowptr) - 1):
            mine = v[rowptr[r]:rowptr[r + 1]]
            p[r] = pow2_of_rows(mine.transpose(1, 0, 2).reshape(16, -1))
        codes, s = quantize_groups(v, gmax, p[brow], fmt)
        return codes, s, p.reshape(-1)
    at = {(r, c): i for i, (r, c) in enumerate(zip(brow.tolist(), colidx.tolist()))}
    both = gmax.copy()
    for (r, c), i in at.items():
        j = at.get((r, c ^ 16))
        if j is not None:
            both[i] = np.maximum(gmax[i], gmax[j])  # NaN if either is
    codes, s = quantize_groups(v, both, 1.0, fmt)
    return codes, s, None


def scale_values(byte, fmt):
    if fmt == "nvfp4":
        return np.where(byte >= 127, np.nan, np.append(E4M3, 0)[np.minimum(byte, 127)])
    return np.where(byte == 255, np.nan, 2.0 ** (byte.astype(np.float64) - 127))


def values(codes, scale_of_code, row):
    """codes and, broadcast against them, scales and row scales -> values in 64 bits."""
    return np.where(codes & 8, -1.0, 1.0) * E2M1[codes & 7] * scale_of_code * row


def dense_values(codes, byte, p, fmt):
    s = np.repeat(scale_values(byte, fmt), GROUP[fmt], axis=1)[:, :codes.shape[1]]
    return values(codes, s, 1.0 if p is None else np.asarray(p, np.float64)[:, None])


def block_values(codes, byte, p, rowptr, fmt):
    brow = np.repeat(np.arange(len(rowptr) - 1), np.diff(rowptr))
    row = 1.0 if p is None else np.asarray(p, np.float64).reshape(-1, 16)[brow][..., None]
    return values(codes, scale_values(byte, fmt)[..., None], row)


def pack(codes):
    """Codes [..., n] -> bytes [..., n / 2], the even one in the low half."""
    return (codes[..., 0::2] | codes[..., 1::2] << 4).astype(np.uint8)


def unpack(b):
    return np.stack([b & 15, b >> 4], -1).reshape(*b.shape[:-1], -1)


def multiply(vals, rowptr, colidx, B):
    """(A x B^T, |A| x |B^T|) of blocks [nnzb, 16, 16] and B [N, K], blocks that are not stored being left out."""
    M, N = (len(rowptr) - 1) * 16, B.shape[0]
    out, mag = np.zeros((M, N)), np.zeros((M, N))
    for r in range(len(rowptr) - 1):
        lo, hi = rowptr[r], rowptr[r + 1]
        if hi > lo:
            k = (colidx[lo:hi, None] + np.arange(16)).reshape(-1)
            a = vals[lo:hi].transpose(1, 0, 2).reshape(16, -1)
            with np.errstate(invalid="ignore"):
                out[r * 16:r * 16 + 16] = a @ B[:, k].T
                mag[r * 16:r * 16 + 16] = np.abs(a) @ np.abs(B[:, k]).T
    return out, mag


def random_blocks(rng, counts, Kb):
    """Block-rows of the given numbers of blocks at random columns -> (rowptr, element columns)."""
    rowptr = np.zeros(len(counts) + 1, np.int32)
    rowptr[1:] = np.cumsum(counts)
    cols = [np.sort(rng.choice(Kb, c, replace=False)) for c in counts]
    return rowptr, (np.concatenate(cols) if cols else np.zeros(0)).astype(np.int32) * 16
