"""CPU restatement (numpy, 64 bits) of the balance loss of expert routers -- TEST INFRASTRUCTURE ONLY: never imported by the
product path.  Written from the definition (no counterpart in the reference): see `balance_losses` in detr_amd/losses.py.
"""
import numpy as np


def chosen_counts(x, top_k, counted, experts=None):
    """[B, E] int64: how often each expert is among a counted row's top_k largest logits (lowest index first among equals,
    never -inf or NaN), or is named by `experts` [B, Q, top_k]."""
    B, Q, E = x.shape
    counts = np.zeros((B, E), dtype=np.int64)
    for b in range(B):
        for q in range(Q):
            if not counted[b, q]:
                continue
            if experts is None:
                row = [(-x[b, q, e], e) for e in range(E) if x[b, q, e] > -np.inf]       # (False for a NaN)
                for _, e in sorted(row)[:top_k]:
                    counts[b, e] += 1
            else:
                for e in experts[b, q]:
                    if 0 <= e < E:
                        counts[b, e] += 1
    return counts


def balance_losses(x, top_k, mask=None, experts=None, counts=None, scores="softmax", per_image=False, grad_balance=None,
                   grad_z=None):
    """One set: x [B, Q, E] float64.  Returns a dict: balance, z, counts (per group: [B] / [B, E], or [1] / [1, E]), grad,
    and what error bounds are made of: p, lse, the shares less one per image (f), 1 / n per image, the rows that count."""
    x = np.asarray(x, dtype=np.float64)
    B, Q, E = x.shape
    counted = ~np.all(x == -np.inf, axis=-1) if Q else np.zeros((B, Q), dtype=bool)
    if mask is not None:
        counted &= mask
    own = chosen_counts(x, top_k, counted, experts)
    rows = counted.sum(1)
    if not per_image:
        own, rows = own.sum(0, keepdims=True), rows.sum(keepdims=True)
    shares_of = own if counts is None else np.asarray(counts).reshape(own.shape)
    total = shares_of.sum(-1, keepdims=True)
    share = np.where(total > 0, E * shares_of / np.maximum(total, 1), 0.0)
    with np.errstate(all="ignore"):
        logs = x if scores == "softmax" else -np.logaddexp(0.0, -x)
        logs = np.where(counted[..., None], logs, 0.0)
        top = logs.max(-1, keepdims=True) if E else logs
        e = np.exp(logs - top)
        lse = (top + np.log(e.sum(-1, keepdims=True)))[..., 0]
        p = np.where(counted[..., None], e / e.sum(-1, keepdims=True), 0.0)        # (exp(logs - lse) fails far from zero)
        lse = np.where(counted, lse, 0.0)
        inv_n = 1.0 / np.maximum(rows, 1)
        group = (lambda v: v.sum(1)) if per_image else (lambda v: v.sum((0, 1), keepdims=True)[0])
        P = group(p) * inv_n[:, None] if per_image else p.sum((0, 1))[None] * inv_n[:, None]
        balance = (share * P).sum(-1)
        z = (lse * lse).sum(1) * inv_n if per_image else (lse * lse).sum(keepdims=True)[0] * inv_n
        f = np.broadcast_to(np.where(total > 0, share - 1.0, 0.0), (B, E))
        per_row = np.broadcast_to(inv_n, (B,))
        gb = np.broadcast_to(0.0 if grad_balance is None else np.asarray(grad_balance, dtype=np.float64).reshape(-1), (B,)) * per_row
        gz = np.broadcast_to(0.0 if grad_z is None else np.asarray(grad_z, dtype=np.float64).reshape(-1), (B,)) * per_row
        dot = (p * f[:, None]).sum(-1, keepdims=True)
        grad = gb[:, None, None] * p * (f[:, None] - dot)
        if scores == "sigmoid":
            grad = grad * np.exp(-np.logaddexp(0.0, x))
        grad = grad + gz[:, None, None] * 2.0 * lse[..., None] * p
        grad = np.where(counted[..., None], grad, 0.0)
    return dict(balance=balance, z=z, counts=own, grad=grad, p=p, lse=lse, f=f, gb=gb, gz=gz, counted=counted)
