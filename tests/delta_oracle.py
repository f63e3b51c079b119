"""The gated delta rule in 64 bits, token by token, and the checks of its results."""
import numpy as np

BF16, F32 = 2, 4


def to_bf16(x):
    """fp32 -> bf16 bit patterns, to the nearest even."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


def forward(q, k, v, g, beta, state, spans, scale, eps):
    """q, k [T, Q, dim], v [T, H, vdim], g, beta [T, H]; spans: (slot, first position, tokens).  Returns out and the states."""
    q, k, v, g, beta = (np.asarray(x, np.float64) for x in (q, k, v, g, beta))
    state = np.array(state, np.float64)
    H, share = v.shape[1], v.shape[1] // q.shape[1]
    if eps > 0:
        q, k = (x / np.sqrt((x * x).sum(-1, keepdims=True) + np.float64(np.float32(eps))) for x in (q, k))
    q, k = np.repeat(q, share, 1), np.repeat(k, share, 1)
    out, t = np.zeros(v.shape), 0
    assert H == k.shape[1]
    for slot, first, n in spans:
        S = np.zeros(state.shape[1:]) if first == 0 else state[slot].copy()
        for _ in range(n):
            S *= np.exp(g[t])[:, None, None]
            u = beta[t][:, None] * (v[t] - np.einsum("hd,hde->he", k[t], S))
            S += k[t][:, :, None] * u[:, None, :]
            out[t] = scale * np.einsum("hd,hde->he", q[t], S)
            t += 1
        state[slot] = S
    return out, state


def inputs(seed, T, Q, H, dim, vdim, elem, slots, unit_keys=False, spread=1.0):
    """Values as a model meets them: heads that forget fast and slowly, tokens that erase more and less."""
    r = np.random.Generator(np.random.PCG64(seed))
    q, k, v = r.normal(size=(T, Q, dim)), r.normal(size=(T, Q, dim)), spread * r.normal(size=(T, H, vdim))
    if unit_keys:
        q, k = (x / np.linalg.norm(x, axis=-1, keepdims=True) for x in (q, k))
    q, k, v = (x.astype(np.float32) for x in (q, k, v))
    if elem == BF16:
        q, k, v = (from_bf16(to_bf16(x)) for x in (q, k, v))
    rate = np.exp(r.uniform(np.log(0.003), np.log(1.5), size=H))
    g = (-rate * np.log1p(np.exp(r.normal(size=(T, H))))).astype(np.float32)
    beta = (1 / (1 + np.exp(-r.normal(size=(T, H))))).astype(np.float32)
    state = (0.3 * r.normal(size=(slots, H, dim, vdim))).astype(np.float32)
    return q, k, v, g, beta, state


def limit(tokens, dim):
    """Largest |difference| of sums in 32 bits over the rms of the wanted values of a head.

    A token's update is a contraction (keys of norm 1 or less, beta below 1), so what rounding puts into a state fades like the state
    itself: its share is at most that of the tokens that are still in it, each of which brings three sums over `dim` terms or 64 tokens
    (fp32 halves of a step, 2^-24, of the largest partial sum).  Independent roundings add up like the root of their number; the largest
    of up to a million values lies within six deviations:  6 * 2^-24 * sqrt(3 dim + min(tokens, 4096)), times 4 for partial sums that
    are larger than their results."""
    return 24 * 2.0 ** -24 * np.sqrt(3 * dim + min(tokens, 4096))


def off(got, want, elem=F32):
    """The largest difference over the rms, by head (axis 1), of the wanted values.  Results in bf16 are rounded once: off by at most
    half a step, 2^-8 of the value itself, however large it is beside the rms; that comes off first."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    axes = (0,) + tuple(range(2, want.ndim))
    rms = np.sqrt((want * want).mean(axes))
    d = np.abs(got - want)
    if elem == BF16:
        d = np.maximum(d - 2.0 ** -8 * np.abs(want), 0.0)
    return float((d.max(axes) / np.maximum(rms, 1e-30)).max())
