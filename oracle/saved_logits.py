"""CPU restatement (numpy, 64 bits) of the classification losses that keep 8 bits per logit -- TEST INFRASTRUCTURE ONLY: never
imported by the product path.  The code is the one include/detr_match.h defines; the losses are those of oracle/cls_loss.py
in 64 bits, their gradients taken at the decoded logits.
"""
import numpy as np

FOCAL_CLAMP, CE_CLAMP = 20.0, 2.0 ** 20
FINEST, FOCAL_COARSEST, CE_COARSEST, NOT_A_NUMBER = -16, -2, -3, -128


def step_exponent(block, coarsest):
    """The finest step of a clamped block (1-D, float64, no NaN)."""
    for e in range(FINEST, coarsest):
        if np.rint(block.max() * 2.0 ** -e) - np.rint(block.min() * 2.0 ** -e) <= 255:
            return e
    return coarsest


def focal_codes(x, keep=True):
    """(bytes [n], heads [blocks], decoded logits like x) of the flat array; the heads as signed 32-bit words.  keep: whether a
    logit's row counts; of the others what lies beyond the clamp, or is NaN, counts as 0.
    """
    flat = np.asarray(x, dtype=np.float64).reshape(-1)
    keep = np.broadcast_to(keep, np.shape(x)).reshape(-1)
    codes, heads, decoded = np.zeros(flat.size, np.uint8), [], np.empty(flat.size)
    for i in range(0, flat.size, 128):
        kept = keep[i:i + 128]
        block = flat[i:i + 128]
        block = np.where(kept, np.clip(block, -FOCAL_CLAMP, FOCAL_CLAMP), np.where(np.abs(block) <= FOCAL_CLAMP, block, 0.0))
        if np.isnan(block).any():
            heads.append(NOT_A_NUMBER & 255)
            decoded[i:i + 128] = np.nan
            continue
        e = step_exponent(block, FOCAL_COARSEST)
        q = np.rint(block * 2.0 ** -e)
        codes[i:i + 128] = q.max() - q
        heads.append(int(q.max()) * 256 + (e & 255))
        decoded[i:i + 128] = q * 2.0 ** e
    return codes, np.array(heads, dtype=np.int64).astype(np.int32), decoded.reshape(np.shape(x))


def ce_codes(x):
    """(bytes [rows, C], steps [rows], decoded logits less the row's largest) of x [rows, C]."""
    x = np.asarray(x, dtype=np.float64)
    codes, steps, decoded = np.zeros(x.shape, np.uint8), np.empty(len(x), np.int8), np.empty(x.shape)
    for r, row in enumerate(x):
        if np.isnan(row).any() or row.max() == np.inf or row.max() == -np.inf:
            steps[r], decoded[r] = NOT_A_NUMBER, np.nan
            continue
        row = np.clip(row, -CE_CLAMP, CE_CLAMP)
        e = step_exponent(row, CE_COARSEST)
        q = np.rint(row * 2.0 ** -e)
        codes[r] = np.minimum(q.max() - q, 255)
        steps[r], decoded[r] = e, -(codes[r].astype(np.float64) * 2.0 ** e)
    return codes, steps, decoded


def focal(x, cls, num_boxes, alpha=0.25, gamma=2.0, ignore_index=None):
    """(loss, grad at the decoded logits for an upstream gradient of one, decoded logits), 64 bits."""
    x = np.asarray(x, dtype=np.float64)
    C = x.shape[-1]
    cls = np.asarray(cls)
    keep = ((cls >= 0) & (cls <= C))[..., None]
    if ignore_index is not None:
        keep = keep & (cls != ignore_index)[..., None]
    hot = cls[..., None] == np.arange(C)
    sign = np.where(hot, -1.0, 1.0)
    factor = (np.where(hot, alpha, 1 - alpha) if alpha >= 0 else 1.0) * keep / num_boxes

    def parts(z):
        return np.logaddexp(0.0, z), np.exp(-np.logaddexp(0.0, -z)), np.exp(-np.logaddexp(0.0, z))

    with np.errstate(all="ignore"):
        softplus, s, _ = parts(sign * x)
        loss = np.where(keep, factor * softplus * s ** gamma, 0.0).sum()
        decoded = focal_codes(x, keep)[2]
        softplus, s, rest = parts(sign * decoded)
        grad = np.where(keep, sign * factor * s ** gamma * (s + gamma * softplus * rest), 0.0)
    return loss, grad, decoded


def cross_entropy(x, cls, weight=None, ignore_index=-100):
    """(loss, grad at the decoded logits for an upstream gradient of one, p), 64 bits, on x [..., C]."""
    shape = np.shape(x)
    x = np.asarray(x, dtype=np.float64).reshape(-1, shape[-1])
    C = x.shape[-1]
    y = np.asarray(cls).reshape(-1)
    keep = (y != ignore_index) & (y >= 0) & (y < C)
    row = np.where(keep, y, 0)
    w = keep * (1.0 if weight is None else np.asarray(weight, dtype=np.float64)[row])
    with np.errstate(all="ignore"):
        top = x.max(-1, keepdims=True)
        lse = (top + np.log(np.exp(x - top).sum(-1, keepdims=True)))[:, 0]
        nll = np.where(w != 0, lse - x[np.arange(len(x)), row], 0.0)
        loss = (w * nll).sum() / w.sum()
        decoded = ce_codes(x)[2]
        e = np.exp(decoded - decoded.max(-1, keepdims=True))
        p = e / e.sum(-1, keepdims=True)
        grad = p - (row[:, None] == np.arange(C))
        grad = np.where((w != 0)[:, None], grad * (w / w.sum())[:, None], 0.0)
    return loss, grad.reshape(shape), p.reshape(shape)
