"""The key/value cache operators restated in 64 bits on the CPU, from their definitions (include/nwc_ops.h)."""
import torch

MIN_NORMAL = 2.0 ** -6                                                # of e4m3


def slot(p, capacity, window, sinks):
    return p if not window or p < sinks else sinks + (p - sinks) % (capacity - sinks)


def rounded_e4m3(y):
    """Nearest e4m3 value (ties to even) of |y| <= 448, in 64 bits."""
    step = torch.exp2(torch.frexp(y.abs().clamp(min=MIN_NORMAL))[1].double() - 4)
    return torch.round(y / step) * step


def unit_exponent(x):
    """Smallest e with max|row| <= 448 * 2^e; -127 for rows of zeros (and never below)."""
    m, e = torch.frexp(x.abs().amax(-1).double())                     # amax = m 2^e, 448 = 0.875 * 2^9
    e = e - 9 + (m > 0.875).int()
    return torch.where(m == 0, torch.full_like(e, -127), e).clamp(min=-127)


def held(codes, byte):
    """Values of e4m3 codes with their rows' exponent bytes."""
    return codes.double() * torch.exp2(byte.double() - 127)[..., None]


def turned(x, norm, cos, sin, eps):
    """x [T, heads, hd] fp64 -> RMSNorm (norm or None) and rotary embedding with rows cos, sin [T, hd]; also the sum of the
    magnitudes that are added up, for error bounds."""
    if norm is not None: x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * norm.double()
    h = x.shape[-1] // 2
    c, s = cos.double()[:, None], sin.double()[:, None]
    rot = torch.cat([-x[..., h:], x[..., :h]], -1)
    return x * c + rot * s, (x * c).abs() + (rot * s).abs()


def attend(q, k, v, pos, window=0, sinks=0, visible=None, depth=None, scale=None):
    """q [T, n_q, hd]; k, v [n_kv, capacity, hd] by slot; all fp64.  Returns (out [T, n_q, hd], sum of p |v| of the same shape)."""
    T, n_q, hd = q.shape
    n_kv, capacity = k.shape[:2]
    scale = hd ** -0.5 if scale is None else scale
    end = pos + T
    at = [p for p in range(end) if not window or p < sinks or p > pos - window]
    slots = torch.tensor([slot(p, capacity, window, sinks) for p in at])
    at = torch.tensor(at)
    sees = torch.zeros(T, len(at), dtype=torch.bool)
    for t in range(T):
        own = pos + (int(depth[t]) if depth is not None else t)
        row = torch.ones(len(at), dtype=torch.bool)
        if window: row = (at < sinks) | (at > own - window)
        if visible is None: row &= at <= own
        else:
            for i, p in enumerate(at.tolist()):
                if p >= pos: j = p - pos; row[i] = bool((int(visible[t, j // 32]) >> (j % 32)) & 1)
        sees[t] = row
    out, weight = torch.zeros(T, n_q, hd, dtype=torch.float64), torch.zeros(T, n_q, hd, dtype=torch.float64)
    for h in range(n_q):
        kv = h // (n_q // n_kv)
        x = (q[:, h] @ k[kv, slots].T) * scale
        for t in range(T):                                            # masked places are left out, whatever they hold
            m = sees[t]
            if not m.any(): continue
            p = torch.softmax(x[t, m], -1)
            out[t, h], weight[t, h] = p @ v[kv, slots[m]], p @ v[kv, slots[m]].abs()
    return out, weight


def tree_bits(T, rows):
    """visible words from per-token lists of seen drafts."""
    words = torch.zeros(T, (T + 31) // 32, dtype=torch.int64)
    for t, seen in enumerate(rows):
        for j in seen: words[t, j // 32] |= 1 << (j % 32)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
