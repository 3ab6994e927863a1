"""numpy restatement, in 64 bits, of attention in a sliding window, attention over a
shared prefix, and rotary positions with several axes."""

import numpy as np


def attend(q, k, v, seen, scale):
    """softmax(scale q k^T) v of each row over the keys that it sees (seen: (rows,
    keys) of booleans); rows that see none are 0.  Nothing else reaches a row.  Also
    the same sum of |v|, and per row the largest sum of |q| |k| over the columns."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    out, size, reach = np.zeros((len(q), v.shape[1])), np.zeros((len(q), v.shape[1])), np.zeros(len(q))
    with np.errstate(all="ignore"):
        if np.isfinite(v).all() and np.isfinite(k).all():
            s = np.where(seen, scale * (q @ k.T), -np.inf)
            top = s.max(1, keepdims=True, initial=-np.inf)
            p = np.exp(s - np.where(np.isneginf(top), 0.0, top))
            total = p.sum(1, keepdims=True)
            p = np.where(total == 0, 0.0, p / np.where(total == 0, 1.0, total))
            out, size = p @ v, p @ np.abs(v)
            reach = np.where(seen, np.abs(q) @ np.abs(k).T, 0.0).max(1, initial=0.0)
        else:
            for i in range(len(q)):
                at = np.flatnonzero(seen[i])
                s = scale * (k[at] @ q[i])
                top = s.max(initial=-np.inf)
                p = np.exp(s - (0.0 if np.isneginf(top) else top))
                if p.sum() == 0:
                    continue
                out[i], size[i] = p @ v[at] / p.sum(), p @ np.abs(v[at]) / p.sum()
                reach[i] = (np.abs(k[at]) @ np.abs(q[i])).max(initial=0.0)
    return out, size, reach


def _cut(lengths, count, most):
    return [most] * count if lengths is None else [max(0, min(most, int(n))) for n in lengths]


def _heads(q, kv_of, seen_of, scale):
    b, hq, sq, d = q.shape
    out, size, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:3])
    for i in range(b):
        seen = seen_of(i)
        for h in range(hq):
            k, v = kv_of(i, h)
            out[i, h], size[i, h], reach[i, h] = attend(q[i, h], k, v, seen, scale)
    return out, size, reach


def sliding_window_attention(q, k, v, window, sinks=0, lengths=None, scale=1.0):
    """(output, the same sum of |v|, per row the largest sum of |q| |k|)"""
    (b, hq, sq, _), (_, hkv, c, _) = q.shape, k.shape
    lengths = _cut(lengths, b, c)
    window, sinks = min(window, c), min(sinks, c)

    def seen(i):
        p = lengths[i] - sq + np.arange(sq)[:, None]
        j = np.arange(c)[None]
        return (j <= p) & ((j > p - window) | (j < sinks))

    return _heads(q, lambda i, h: (k[i, h // (hq // hkv)], v[i, h // (hq // hkv)]), seen, scale)


def shared_prefix_attention(q, pk, pv, k, v, prefix_lengths=None, lengths=None, scale=1.0):
    (b, hq, sq, _), (_, hkv, c, _), (g, _, p, _) = q.shape, k.shape, pk.shape
    lengths, prefix_lengths = _cut(lengths, b, c), _cut(prefix_lengths, g, p)

    def seen(i):
        own = np.arange(c)[None] <= lengths[i] - sq + np.arange(sq)[:, None]
        front = np.arange(p) < prefix_lengths[i // (b // g)]
        return np.concatenate((np.broadcast_to(front, (sq, p)), own), 1)

    def kv(i, h):
        of, hk = i // (b // g), h // (hq // hkv)
        return np.concatenate((pk[of, hk], k[i, hk])), np.concatenate((pv[of, hk], v[i, hk]))

    return _heads(q, kv, seen, scale)


def multi_axis_rotary_position_embedding(x, sin, cos, positions, sections, interleaved):
    """x (batch, seq, heads, dim); positions (axes, batch, seq)."""
    axes, (dim, half) = len(positions), (x.shape[-1], x.shape[-1] // 2)
    first = [2 * i if interleaved else i for i in range(half)]
    second = [2 * i + 1 if interleaved else i + half for i in range(half)]
    axis = [s % axes for s, n in enumerate(sections) for _ in range(n)]
    out = np.zeros(x.shape)
    for i in range(half):
        row = positions[axis[i]]
        inside = (row >= 0) & (row < len(sin))
        at = np.where(inside, row, 0)
        wide = sin.shape[1] == dim
        for e, other, sign in ((first[i], second[i], -1.0), (second[i], first[i], 1.0)):
            col = e if wide else i
            s, c = (np.where(inside, t[at, col] if len(t) else 0.0, np.nan)[..., None] for t in (sin, cos))
            out[..., e] = x[..., e] * c + sign * x[..., other] * s
    return out
