"""AdamW over many tensors in float64 numpy, one tensor at a time, from the formulas; the 8-bit moments by a table of the codes'
values.  What the GPU tests of pde_amd.optim.GroupedAdamW compare with; nothing here is the framework's code."""
import numpy as np

BLOCK = 128
M = dict(bias=7, codes=127, most=246, place=0x9E3779B9, step=0xC13FA9A9)
V = dict(bias=15, codes=255, most=238, place=0x6A09E667, step=0x91E10DA5)


def table(form):
    return np.array([c / 8 * 2.0 ** (1 - form["bias"]) if c < 8 else (1 + c % 8 / 8) * 2.0 ** (c // 8 - form["bias"]) for c in range(form["codes"])])


def values(code, scale, form):
    """flat codes and their blocks' scales -> float64"""
    code = np.asarray(code).astype(np.int64)
    tab = table(form)
    if form is M:
        x = np.where(code >= 128, -1.0, 1.0) * tab[code % 128]
    else:
        x = tab[code]
    s = np.repeat(np.asarray(scale).astype(np.int64), BLOCK)
    return np.where(s == 255, np.nan, x * 2.0 ** (np.minimum(s, 254) - 127.0))


def round_block(x, first, t, form):
    """one block (128 values, the first at place `first` of the layout) -> (values, scale byte)"""
    if not np.isfinite(x).all():
        return np.full(x.shape, np.nan), 255
    tab = table(form)
    a = np.abs(x)
    scale = 0
    while scale < form["most"] and a.max() >= tab[-1] * 2.0 ** (scale - 127):
        scale += 1
    y = a * 2.0 ** (127 - scale)
    c = np.clip(np.searchsorted(tab, y, side="right") - 1, 0, len(tab) - 2)
    i = np.arange(first, first + len(x), dtype=np.uint64)
    word = (i * np.uint64(form["place"]) + np.uint64(t * form["step"] % 2 ** 32)) % np.uint64(2 ** 32)
    u = ((word >> np.uint64(15)) | np.uint64(1)).astype(np.float64) / 2 ** 17
    place = c + (y - tab[c]) / (tab[c + 1] - tab[c])                           # on the codes' own scale, a float64: rounded once
    c = np.floor(place + u).astype(np.int64)
    if form is V:
        c = np.where(a > 0, np.maximum(c, 1), c)
    return np.where(x < 0, -1.0, 1.0) * tab[c] * 2.0 ** (scale - 127), scale


def round_flat(x, offset, t, form):
    """a tensor's moments (float64, flat, at `offset` of the layout) as they are held in 8 bits, and the scales of its blocks"""
    n = len(x)
    pad = np.zeros(-n % BLOCK)
    x = np.concatenate([x, pad])
    out, scales = np.empty_like(x), []
    for b in range(0, len(x), BLOCK):
        out[b:b + BLOCK], s = round_block(x[b:b + BLOCK], offset + b, t, form)
        scales.append(s)
    return out[:n], np.array(scales, dtype=np.uint8)


def clip_factor(grads, max_norm):
    norm = np.sqrt(sum(float((np.asarray(g, dtype=np.float64) ** 2).sum()) for g in grads))
    f = max_norm / (norm + 1e-6)
    return norm, (1.0 if f > 1.0 else f)


def step(p, g, m, v, t, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=1e-2):
    """one tensor, float64: (p, m, v) after step t"""
    p, g, m, v = (np.asarray(x, dtype=np.float64) for x in (p, g, m, v))
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    with np.errstate(invalid="ignore", divide="ignore"):
        p = p * (1 - lr * wd) - lr / (1 - b1 ** t) * m / (np.sqrt(v / (1 - b2 ** t)) + eps)
    return p, m, v
