"""The rules on logits in NumPy float32, one operation at a time (the kernel's
order and roundings)."""
import numpy as np


def reference(x, hist=None, hist_off=None, repetition=None, presence=None, frequency=None,
              bias_id=None, bias_val=None, bias_off=None, mask=None, mask_row=None):
    """x float32 [M][V]; lists as NumPy arrays or None."""
    y = np.array(x, np.float32)
    M, V = y.shape
    f = np.float32

    def span(off, r, n):
        b = min(max(int(off[r]), 0), n)
        return b, min(max(int(off[r + 1]), b), n)

    with np.errstate(all="ignore"):
        for r in range(M):
            if hist is not None:
                b, e = span(hist_off, r, len(hist))
                ids, counts = np.unique(hist[b:e], return_counts=True)
                ok = (ids >= 0) & (ids < V)
                ids, c = ids[ok], counts[ok].astype(f)
                rep = f(1) if repetition is None else f(repetition[r])
                pres = f(0) if presence is None else f(presence[r])
                freq = f(0) if frequency is None else f(frequency[r])
                v = y[r, ids]
                v = np.where(v > 0, v / rep, v * rep)
                y[r, ids] = v - (pres + freq * c)
            if bias_id is not None:
                b, e = span(bias_off, r, len(bias_id))
                last = dict(zip(bias_id[b:e].tolist(), bias_val[b:e].tolist()))
                for j, w in last.items():
                    if 0 <= j < V:
                        y[r, j] = y[r, j] + f(w)
            if mask is not None:
                k = r if mask_row is None else int(mask_row[r])
                if 0 <= k < len(mask):
                    j = np.arange(V)
                    bits = (mask[k].view(np.uint32)[j // 32] >> (j % 32).astype(np.uint32)) & 1
                    y[r, bits == 0] = -np.inf
    return y


def words(allowed):
    """Bool [n][V] as mask words int32 [n][ceil(V / 32)]."""
    n, V = allowed.shape
    pad = np.zeros((n, (V + 31) // 32 * 32), bool)
    pad[:, :V] = allowed
    return np.packbits(pad, axis=1, bitorder="little").view(np.uint32).view(np.int32).reshape(n, -1)
